"""The clipped policy loss over sampled answers against its definition in 64 bits.

Tolerances, of norms: bfloat16 gradients are one rounding (half a step, 2^-8). 32-bit: a
probability is an exponential (hardware, 2^-22, and its argument's rounding, up to 2^-24 * 40) over
a sum of at most 2^18 in threads and trees (20 roundings): 3e-6 one way; gradients are differences of
a few such terms of the same size: 1e-5. Log-probabilities are taken in 64 bits from that sum: 1e-6 of
their norm; the loss is held to 1e-5 of the sum of its terms' sizes.
"""
import pytest
import torch

from surfb200.ops import _lib, gemm as G, rl as R, tokens as TK

pytestmark = pytest.mark.gpu
BF, F32 = torch.bfloat16, torch.float32


def rel(x, y):
    y = y.detach().double()
    n = float(torch.linalg.vector_norm(y))
    return float(torch.linalg.vector_norm(x.double() - y)) / (n if n else 1.0)


def make(rows, v, dtype, seed=0, masked=True, clip=0.2):
    gen = torch.Generator("cuda").manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=gen, device="cuda")  # noqa: E731
    z = 2 * r(rows, v)
    a = torch.randint(0, v, (rows,), generator=gen, device="cuda", dtype=torch.int32)
    if masked and v > 3:
        z[torch.rand(rows, v, generator=gen, device="cuda") < 0.1] = float("-inf")
        z[torch.rand(rows, v, generator=gen, device="cuda") < 0.02] = float("nan")
        if rows > 3:
            a[1], a[2] = -1, -7
            z[3] = float("-inf")
    z = z.to(dtype)
    zd = torch.where(z.isnan(), torch.full_like(z, float("-inf")), z).double()
    lp = torch.nan_to_num(torch.log_softmax(zd, 1).gather(1, a.long().clamp(min=0)[:, None])[:, 0], nan=0.0, neginf=-3.0).float()
    moved = 0.3 * r(rows)
    near = ((torch.exp(moved) - 1).abs() - clip).abs() < 1e-2          # not where 32 bits may clip another way
    return dict(logits=z, answers=a, old_logp=lp - torch.where(near, 0.5 * moved, moved), advantages=r(rows), ref_logp=lp + 0.3 * r(rows),
                weights=torch.rand(rows, generator=gen, device="cuda") / rows)


def oracle(c, **kw):
    z = torch.where(c["logits"].isnan(), torch.full_like(c["logits"], float("-inf")), c["logits"]).double().requires_grad_()
    d = {k: None if c.get(k) is None else c[k].double() for k in ("old_logp", "advantages", "ref_logp", "weights")}
    loss = R.policy_loss_reference(z, c["answers"], d["old_logp"], d["advantages"], ref_logp=d["ref_logp"], weights=d["weights"], **kw)
    return loss.detach(), torch.nan_to_num(torch.autograd.grad(loss, z)[0])


def call(c, **kw):
    return R.policy_loss(c["logits"], c["answers"], c["old_logp"], c["advantages"], ref_logp=c.get("ref_logp"),
                         weights=c.get("weights"), **kw)


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("rows,v", [(1, 1), (5, 2), (33, 15), (40, 32), (9, 100), (70, 511), (6, 513), (150, 1000), (3, 8191), (4, 32003),
                                    (200, 5000), (2, 131072), (2, 262144)])
def test_against_the_definition(rows, v, dtype):
    c = make(rows, v, dtype)
    kw = dict(kl_coef=0.1, ent_coef=0.02, temperature=1.0)
    loss, grad = oracle(c, **kw)
    r = call(c, **kw)
    half = torch.finfo(dtype).eps / 2 if dtype == BF else 0.0
    size = float((c["weights"].double().abs() * (1 + c["advantages"].abs())).sum())
    assert abs(float(r.loss) - float(loss)) < 1e-5 * size
    assert rel(r.dlogits, grad) < half + 1e-5
    z = torch.where(c["logits"].isnan(), torch.full_like(c["logits"], float("-inf")), c["logits"]).double()
    at = c["answers"].long().clamp(min=0)[:, None]
    on = (c["answers"] >= 0) & (z.gather(1, at)[:, 0] > float("-inf"))
    logp = torch.log_softmax(torch.where(on[:, None], z, torch.zeros_like(z)), 1)
    lp = torch.where(on, logp.gather(1, at)[:, 0], 0.0)
    ent = torch.where(on, -torch.nan_to_num(logp.exp() * logp, nan=0.0).sum(1), 0.0)
    d = c["ref_logp"].double() - lp
    assert rel(r.logp, lp) < 1e-6 and rel(r.entropy, ent) < 1e-5
    assert rel(r.kl, torch.where(on, torch.exp(d) - d - 1, 0.0)) < 1e-5
    assert not r.dlogits[~on].any()


@pytest.mark.parametrize("v", [12, 700])
@pytest.mark.parametrize("kw", [dict(), dict(temperature=0.5), dict(clip=0.1, clip_high=0.4), dict(ent_coef=0.1), dict(kl_coef=1.0, temperature=2.0)])
def test_options(v, kw):
    c = make(64, v, F32, clip=kw.get("clip", 0.2))
    if kw.get("temperature") or kw.get("clip_high"):
        # log-probabilities of the other temperature, ratios on one side of both borders
        zd = torch.where(c["logits"].isnan(), torch.full_like(c["logits"], float("-inf")), c["logits"]).double()
        lp = torch.nan_to_num(torch.log_softmax(zd / kw.get("temperature", 1.0), 1).gather(1, c["answers"].long().clamp(min=0)[:, None])[:, 0],
                              nan=0.0, neginf=-3.0).float()
        moved = torch.linspace(-0.8, 0.83, 64, device="cuda")
        c["old_logp"], c["ref_logp"] = lp - moved, lp + 0.2
    if "kl_coef" not in kw:
        c["ref_logp"] = None
    c["weights"] = None
    loss, grad = oracle(c, **kw)
    r = call(c, **kw)
    assert abs(float(r.loss) - float(loss)) < 1e-5 * float(1 + c["advantages"].abs().mean())
    assert rel(r.dlogits, grad) < 1e-5
    n = call(c, grad=False, **kw)
    assert n.dlogits is None and torch.equal(n.loss, r.loss) and torch.equal(n.logp, r.logp)


def test_gradient_by_differences():
    c = make(6, 9, F32, masked=False)
    kw = dict(kl_coef=0.3, ent_coef=0.1, temperature=0.8)
    got = call(c, **kw).dlogits.double()
    z = c["logits"].double()
    h = 1e-6
    for i, j in ((0, 0), (1, int(c["answers"][1])), (5, 8)):
        d = [float(oracle(dict(c, logits=z + s * h * torch.zeros_like(z).index_put((torch.tensor(i), torch.tensor(j)), torch.tensor(1.0, dtype=torch.float64, device="cuda"))), **kw)[0])
             for s in (1, -1)]
        assert abs((d[0] - d[1]) / (2 * h) - float(got[i, j])) < 1e-6


def test_infinite_logits_share_the_probability():
    for v in (20, 900):
        c = make(4, v, F32, masked=False)
        c["logits"][:, [2, 7]] = float("inf")
        c["answers"][:] = torch.tensor([2, 7, 2, 7], dtype=torch.int32)
        r = call(c, ent_coef=0.1)
        torch.testing.assert_close(r.logp, torch.full((4,), -0.6931472, device="cuda"))
        torch.testing.assert_close(r.entropy, torch.full((4,), 0.6931472, device="cuda"))
        assert torch.isfinite(r.dlogits).all() and not r.dlogits[:, 8:].any()


@pytest.mark.parametrize("size", [1e3, 5e5, 7.3e5, 1e6, 1e8, 1e30])
def test_large_logits(size):
    """Logits of any size about each other: their differences are what counts. A log-probability is a
    difference of numbers of that size, each exact, times 1 / t in 32 bits (2^-24 of the difference)."""
    for v in (40, 3000, 140000):
        gen = torch.Generator("cuda").manual_seed(5)
        z = torch.randn(3, v, generator=gen, device="cuda") * min(2.0, 1e-7 * size + 1.0) + size
        z[1] = -z[1]
        z[2, ::2] = -size
        a = z.argmax(1).to(torch.int32)
        a[0] = 1
        c = dict(logits=z, answers=a, old_logp=torch.zeros(3, device="cuda"), advantages=torch.ones(3, device="cuda"))
        r = R.policy_loss(**c, ent_coef=0.1, clip=1.0, clip_high=1e30)
        zd = z.double().requires_grad_()
        want = R.policy_loss_reference(zd, a, c["old_logp"].double(), c["advantages"].double(), ent_coef=0.1, clip=1.0, clip_high=1e30)
        lp = torch.log_softmax(zd.detach(), 1).gather(1, a.long()[:, None])[:, 0]
        assert rel(r.logp, lp) < 1e-6
        assert rel(r.dlogits, torch.autograd.grad(want, zd)[0]) < 1e-5


def test_far_ratios():
    """A ratio of e^200 is infinite in 32 bits: its loss is, no advantage means no loss; small ones vanish."""
    c = make(4, 10, F32, masked=False)
    c["ref_logp"] = None
    lp = call(c).logp
    c["old_logp"] = lp + torch.tensor([200.0, -200.0, -200.0, 200.0], device="cuda")
    c["advantages"] = torch.tensor([1.0, 1.0, 0.0, -1.0], device="cuda")
    r = call(c)
    assert torch.isfinite(r.dlogits).all() and torch.isfinite(r.loss)
    assert not r.dlogits[1:].any()


@pytest.mark.parametrize("v", [30, 1001])
@pytest.mark.parametrize("dtype", [BF, F32])
def test_strides_in_place_and_answers_of_64_bits(v, dtype):
    c = make(37, v, dtype)
    kw = dict(kl_coef=0.1, ent_coef=0.01)
    want = call(c, **kw)
    wide = torch.full((37, v + 13), 7.0, dtype=dtype, device="cuda")
    wide[:, 5:5 + v] = c["logits"]
    view = wide[:, 5:5 + v]
    other = dict(c, logits=view, answers=c["answers"].long())
    half = torch.finfo(dtype).eps if dtype == BF else 0.0
    r = call(other, **kw)
    assert rel(r.dlogits, want.dlogits) < half + 1e-6 and rel(r.logp, want.logp) < 1e-6
    out = torch.empty(37, v + 1, dtype=dtype, device="cuda")[:, 1:]
    assert torch.equal(call(other, out=out, **kw).dlogits, r.dlogits)
    assert call(other, out=view, **kw).dlogits is view
    assert torch.equal(view, r.dlogits)
    assert bool((wide[:, :5] == 7.0).all()) and bool((wide[:, 5 + v:] == 7.0).all())


def test_offsets_past_32_bits():
    for v in (20, 2000):
        c = make(2, v, BF, masked=False)
        want = call(c)
        big = torch.empty(2 ** 32 + v, dtype=BF, device="cuda")
        far = torch.as_strided(big, (2, v), (2 ** 32, 1))
        far.copy_(c["logits"])
        assert torch.equal(call(dict(c, logits=far), out=far).dlogits, want.dlogits)


def test_answer_past_the_row_is_reported():
    for v in (30, 1000):
        c = make(5, v, F32)
        c["answers"][4] = v
        G.check_error_flag("cuda")
        r = call(c)
        assert not r.dlogits[4].any() and float(r.logp[4]) == 0.0
        with pytest.raises(_lib.KernelError, match="loss sample"):
            G.check_error_flag("cuda")


def test_streams_graphs_and_no_rows():
    for v in (30, 3000):
        c = make(50, v, BF)
        want = call(c, kl_coef=0.1)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            other = call(c, kl_coef=0.1)
        here = call(c, kl_coef=0.1)
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            replayed = call(c, kl_coef=0.1)
        graph.replay()
        torch.cuda.synchronize()
        for r in (other, here, replayed):
            for x, y in zip(r, want):
                assert torch.equal(x, y)
    c = make(0, 9, F32, masked=False)
    assert float(call(c).loss) == 0.0


def test_sampled_answers_train_their_policy():
    """Answers drawn by sample_tokens, their log-probabilities as old_logp: ratios are 1, and the gradient
    is the plain policy gradient."""
    gen = torch.Generator("cuda").manual_seed(3)
    z = torch.randn(64, 40, generator=gen, device="cuda")
    tok, logp = TK.sample_tokens(z, torch.rand(64, 1, generator=gen, device="cuda"), temperature=0.7)
    adv = torch.randn(64, generator=gen, device="cuda")
    r = R.policy_loss(z, tok[:, 0].contiguous(), logp[:, 0].contiguous(), adv, temperature=0.7)
    assert rel(r.logp, logp[:, 0]) < 1e-5
    p = torch.softmax(z.double() / 0.7, 1)
    want = -(adv.double() / 64)[:, None] * (torch.nn.functional.one_hot(tok[:, 0].long(), 40) - p) / 0.7
    assert rel(r.dlogits, want) < 1e-5


def test_refusals():
    c = make(4, 20, F32)
    with pytest.raises(ValueError, match="logits must be"):
        call(dict(c, logits=c["logits"][0]))
    with pytest.raises(TypeError, match="bfloat16 or float32"):
        call(dict(c, logits=c["logits"].half()))
    with pytest.raises(ValueError, match="candidates"):
        call(dict(c, logits=torch.zeros(4, 262145, device="cuda")))
    with pytest.raises(ValueError, match="dense last axis"):
        call(dict(c, logits=c["logits"].t().contiguous().t()))
    with pytest.raises(TypeError, match="answers must be"):
        call(dict(c, answers=c["answers"].float()))
    with pytest.raises(ValueError, match="answers must be"):
        call(dict(c, answers=c["answers"][:3]))
    with pytest.raises(ValueError, match="old_logp"):
        call(dict(c, old_logp=c["old_logp"].double()))
    with pytest.raises(ValueError, match="weights"):
        call(dict(c, weights=c["weights"].cpu()))
    for bad in (dict(clip=-0.1), dict(clip=float("nan")), dict(clip=1.5), dict(clip_high=-1.0), dict(temperature=0.0), dict(temperature=float("nan")),
                dict(kl_coef=float("inf")), dict(ent_coef=float("nan"))):
        with pytest.raises(ValueError):
            call(c, **bad)
    with pytest.raises(ValueError, match="out without grad"):
        call(c, grad=False, out=torch.empty_like(c["logits"]))
    with pytest.raises(ValueError, match="out must be like"):
        call(c, out=torch.empty(4, 20, dtype=BF, device="cuda"))
    with pytest.raises(ValueError, match="shares memory"):
        call(c, out=torch.as_strided(c["logits"], (4, 20), (19, 1)))
    with pytest.raises(_lib.KernelError):
        R.policy_loss(*(c[k].cpu() for k in ("logits", "answers", "old_logp", "advantages")))


def test_numbers_past_float32_and_rows_that_share_memory_are_refused():
    c = make(4, 20, F32)
    for bad in (dict(clip_high=1e39), dict(temperature=1e-39), dict(temperature=1e39), dict(kl_coef=1e39), dict(ent_coef=-1e300)):
        with pytest.raises(ValueError):
            call(c, **bad)
    with pytest.raises(ValueError, match="share memory"):
        call(c, out=torch.zeros(80, device="cuda").as_strided((4, 20), (10, 1)))
    rows = torch.zeros(80, device="cuda").as_strided((4, 20), (10, 1))
    with pytest.raises(ValueError, match="share memory"):
        call(dict(c, logits=rows), out=rows)


def test_two_calls_at_once():
    # the same rows on two streams, neither waiting for the other
    for v, dtype in ((15, F32), (700, BF), (60000, BF)):
        c = make(64, v, dtype)
        want = call(c, kl_coef=0.1)
        torch.cuda.synchronize()
        streams, got = [torch.cuda.Stream() for _ in range(2)], []
        for s in streams * 4:
            with torch.cuda.stream(s):
                got.append(call(c, kl_coef=0.1))
        torch.cuda.synchronize()
        for r in got:
            assert torch.equal(r.loss, want.loss) and torch.equal(r.dlogits, want.dlogits) and torch.equal(r.logp, want.logp)
