"""The answer sampler against its rule by sorting: the same answers (whole numbers of
weight make every sum exact, so they are equal, not close), log-probabilities to two
roundings of 32 bits; empty rows, ties, infinities, NaN, limits per row; frequencies."""
import pytest
import torch

from surfb200.models.policy import HeadLayout
from surfb200.ops import _lib
from surfb200.ops import tokens as TK

pytestmark = pytest.mark.gpu


def _same(logits, u, **kw):
    tok, logp = TK.sample_tokens(logits, u, **kw)
    # the rule's exponential on the same device, so that weights are the same numbers
    et, ep = _by_rule(logits, u, **kw)
    assert torch.equal(tok, et)
    assert torch.allclose(logp, ep, rtol=2.0 ** -22, atol=1e-6)
    assert torch.equal(torch.isinf(logp), tok < 0)
    return tok, logp


def _by_rule(logits, u, **kw):
    """sample_tokens_reference with the exponentials of the GPU."""
    keep = torch.exp

    def gpu_exp(x):
        return keep(x.cuda()).cpu() if x.dtype == torch.float32 else keep(x)

    torch.exp = gpu_exp
    try:
        cpu = {k: v.cpu() if isinstance(v, torch.Tensor) else v for k, v in kw.items()}
        t, p = TK.sample_tokens_reference(logits.cpu(), u.cpu(), **cpu)
    finally:
        torch.exp = keep
    return t.cuda(), p.cuda()


RULES = [dict(), dict(top_k=1), dict(top_k=5), dict(top_p=0.9), dict(top_p=0.5, top_k=40), dict(min_p=0.1),
         dict(temperature=0.0), dict(temperature=0.3, top_p=0.99, min_p=0.01), dict(temperature=3.0, top_k=1000, top_p=0.7),
         dict(top_p=0.0), dict(min_p=1.0)]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("rule", RULES, ids=str)
@pytest.mark.parametrize("rows,vocab", [(5, 2), (7, 31), (3, 33), (4, 1000), (2, 8193), (1, 40001)])
def test_equals_the_rule(rows, vocab, rule, dtype):
    gen = torch.Generator("cuda").manual_seed(rows * vocab)
    z = (3 * torch.randn(rows, vocab + 3, generator=gen, device="cuda")).to(dtype)[:, 1:vocab + 1]
    z[torch.rand(rows, vocab, generator=gen, device="cuda") < 0.1] = float("-inf")
    u = torch.rand(rows, 1, generator=gen, device="cuda")
    _same(z, u, **rule)


@pytest.mark.parametrize("vocab", [9, 3000, 20000, 131072])
def test_ties_go_to_the_lowest_index(vocab):
    z = torch.zeros(4, vocab, device="cuda")
    z[1, vocab // 2:] = -0.0                                    # equal to +0
    z[2] = torch.arange(vocab, device="cuda") % 3
    z[3, :vocab // 2] = -1.0
    for rule in (dict(top_k=4), dict(top_p=0.25), dict(top_k=vocab // 2 + 1, top_p=0.5), dict(temperature=0.0), dict()):
        for q in (0.0, 0.37, 0.9999):
            _same(z, torch.full((4, 1), q, device="cuda"), **rule)
    tok, _ = TK.sample_tokens(z, torch.full((4, 1), 0.9999, device="cuda"), top_k=2)
    assert tok[:, 0].tolist() == [1, 1, 5, vocab // 2 + 1]


@pytest.mark.parametrize("vocab", [20, 5000])
def test_empty_rows_infinities_and_nan(vocab):
    inf = float("inf")
    z = torch.zeros(6, vocab, device="cuda")
    z[0] = -inf
    z[1] = float("nan")
    z[2, :] = -inf
    z[2, 7] = torch.finfo(torch.float32).min                     # the only candidate
    z[3, 3] = z[3, 9] = inf                                      # share everything
    z[4, ::2] = float("nan")
    z[5] = torch.finfo(torch.float32).min                        # masked by the lowest value: all equal
    for rule in (dict(), dict(top_k=3), dict(top_p=0.9), dict(top_k=3, top_p=0.4, min_p=0.2)):
        tok, logp = _same(z, torch.full((6, 1), 0.6, device="cuda"), **rule)
        assert tok[:3, 0].tolist() == [-1, -1, 7] and logp[2, 0] == 0
        assert tok[3, 0] in (3, 9) and tok[4, 0] % 2 == 1


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_many_long_rows(dtype):
    """As many rows as there are blocks to run them, each one block's: ordinary ones, ties,
    empty ones, an odd offset."""
    gen = torch.Generator("cuda").manual_seed(3)
    n, vocab = 150, 9001
    wide = (2.5 * torch.randn(n, vocab + 6, generator=gen, device="cuda")).to(dtype)
    wide[0] = 0.0
    wide[1] = float("-inf")
    wide[2, 5000:] = float("nan")
    wide[3, ::2] = 7.0
    wide[4] = (torch.arange(vocab + 6, device="cuda") % 5).to(dtype)
    z = wide[:, 3:vocab + 3]
    u = torch.rand(n, 1, generator=gen, device="cuda")
    for rule in (dict(), dict(top_p=0.9), dict(top_k=30, top_p=0.8), dict(top_k=4600, min_p=1e-4), dict(top_k=7000, top_p=0.99),
                 dict(temperature=0.0)):
        _same(z, u, **rule)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_many_long_rows_under_a_count(dtype):
    """Most candidates far below the limit: one kept per row, infinite ones, a limit on the
    boundary of two equal ones, per-row limits of which some are none."""
    gen = torch.Generator("cuda").manual_seed(4)
    n, vocab = 149, 12345
    z = torch.randn(n, vocab, generator=gen, device="cuda").to(dtype)
    z[0, 77] = z[0, 9000] = float("inf")
    z[1, 1:] = float("-inf")
    z[2, 12344] = 30.0
    z[3, 5:8] = 20.0
    z[4] = -1000.0
    z[4, 128:256] = 1000.0
    u = torch.rand(n, 1, generator=gen, device="cuda")
    k = torch.arange(n, device="cuda", dtype=torch.int32) % 7
    for rule in (dict(top_k=2), dict(top_k=k), dict(top_k=k, temperature=0.05), dict(top_k=64, top_p=0.5, min_p=0.01),
                 dict(top_k=12000)):
        _same(z, u, **rule)


def test_limits_per_row():
    gen = torch.Generator("cuda").manual_seed(1)
    z = 2 * torch.randn(8, 700, generator=gen, device="cuda")
    u = torch.rand(8, 1, generator=gen, device="cuda")
    r = torch.arange(8, device="cuda")
    _same(z, u, temperature=0.2 * r.float(), top_k=(r * 3).int(), top_p=1 - 0.1 * r.float(), min_p=0.02 * r.float())


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_heads(dtype):
    layout = HeadLayout()
    gen = torch.Generator("cuda").manual_seed(2)
    z = torch.randn(300, 64, generator=gen, device="cuda").to(dtype)
    u = torch.rand(300, len(layout.sizes), generator=gen, device="cuda")
    for rule in RULES:
        tok, _ = _same(z, u, heads=layout.sizes, **rule)
        assert (tok < torch.tensor(layout.sizes, device="cuda")).all()
    big = torch.randn(3, 200, generator=gen, device="cuda").to(dtype)
    _same(big, u[:3, :3].contiguous(), heads=(100, 1, 60), top_p=0.8)


def test_offsets_past_32_bits():
    far = (1 << 31) + 4
    buf = torch.zeros(far + 20000, dtype=torch.bfloat16, device="cuda")
    for vocab in (30, 20000):
        z = buf.as_strided((2, vocab), (far, 1))
        z.copy_(torch.randn(2, vocab, device="cuda"))
        u = torch.rand(2, 1, device="cuda")
        a, b = TK.sample_tokens(z, u, top_p=0.9), TK.sample_tokens(z.contiguous(), u, top_p=0.9)
        assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


def test_numbers_at_the_ends():
    z = torch.randn(1, 100, device="cuda").expand(4, 100)
    u = torch.tensor([[0.0], [1.0 - 2.0 ** -24], [1.0], [-1.0]], device="cuda")
    tok, _ = TK.sample_tokens(z, u)
    assert tok[:, 0].tolist() == [0, 99, 99, 0]


def test_frequencies():
    """200,000 draws of 50 answers under top-p: each count within 6 standard deviations
    (a chance of about 1e-7 for all of them)."""
    gen = torch.Generator("cuda").manual_seed(5)
    z = 1.5 * torch.randn(50, generator=gen, device="cuda")
    n = 200_000
    tok, logp = TK.sample_tokens(z.expand(n, 50), torch.rand(n, 1, generator=gen, device="cuda"), temperature=0.9, top_p=0.9)
    p = torch.softmax(z.double() / 0.9, 0)
    order = torch.argsort(p, descending=True)
    kept = torch.zeros(50, dtype=torch.bool, device="cuda")
    kept[order] = (p[order].cumsum(0) - p[order]) < 0.9
    q = torch.where(kept, p, 0.0) / p[kept].sum()
    count = torch.bincount(tok[:, 0].long(), minlength=50).double()
    assert ((count - n * q).abs() <= 6 * (n * q * (1 - q)).sqrt() + 1e-9).all()
    assert torch.allclose(logp[:, 0].double(), q[tok[:, 0].long()].log(), atol=1e-5)


def test_outputs_in_place_and_refusals():
    z = torch.randn(3, 40, device="cuda")
    u = torch.rand(3, 1, device="cuda")
    out = torch.empty(3, 1, dtype=torch.int32, device="cuda")
    logp = torch.empty(3, 1, device="cuda")
    a, b = TK.sample_tokens(z, u, out=out, logp=logp)
    assert a is out and b is logp
    assert TK.sample_tokens(z[:0], u[:0])[0].shape == (0, 1)
    with pytest.raises(_lib.KernelError):
        TK.sample_tokens(z.cpu(), u.cpu())
    with pytest.raises(TypeError, match="bfloat16 or float32"):
        TK.sample_tokens(z.half(), u)
    with pytest.raises(ValueError, match="u must be"):
        TK.sample_tokens(z, u[:2])
    with pytest.raises(ValueError, match="dense last axis"):
        TK.sample_tokens(z.t(), torch.rand(40, 1, device="cuda"))
    with pytest.raises(ValueError, match="heads"):
        TK.sample_tokens(z, u, heads=(41,))
    with pytest.raises(ValueError, match="negative"):
        TK.sample_tokens(z, u, top_p=1.5)
    with pytest.raises(ValueError, match="top_k must be"):
        TK.sample_tokens(z, u, top_k=torch.ones(3, device="cuda"))
    with pytest.raises(ValueError, match="at most"):
        TK.sample_tokens(torch.empty(1, TK.MAX_VOCAB + 1, device="cuda"), u[:1])


def test_outputs_apart_from_inputs():
    """Outputs over the numbers, the logits, a limit or one another are refused; beside them in
    one buffer they are taken."""
    z = torch.randn(3, 40000, device="cuda")
    u, t = torch.rand(3, 1, device="cuda"), torch.ones(3, device="cuda")
    k = torch.full((3,), 9, dtype=torch.int32, device="cuda")
    for kw in (dict(logp=u), dict(out=u.view(torch.int32)), dict(logp=t.view(3, 1), temperature=t), dict(out=k.view(3, 1), top_k=k),
               dict(logp=z[0, 8:11].view(3, 1))):
        with pytest.raises(ValueError, match="memory with"):
            TK.sample_tokens(z, u, **kw)
    both = torch.zeros(3, 1, device="cuda")
    with pytest.raises(ValueError, match="out shares memory with logp"):
        TK.sample_tokens(z, u, out=both.view(torch.int32), logp=both)
    buf = torch.zeros(9, device="cuda")
    buf[3:6] = u[:, 0]
    a = TK.sample_tokens(z, buf[3:6].view(3, 1), out=buf[:3].view(torch.int32).view(3, 1), logp=buf[6:].view(3, 1))
    b = TK.sample_tokens(z, u)
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


@pytest.mark.parametrize("rule", ["temperature", "top_p", "min_p"])
def test_a_rule_that_is_not_a_number_is_refused(rule):
    z, u = torch.randn(3, 40, device="cuda"), torch.rand(3, 1, device="cuda")
    with pytest.raises(ValueError, match="negative"):
        TK.sample_tokens(z, u, **{rule: float("nan")})


def _same_in(rows, logits, u, **kw):
    """``_same`` for a few of the rows of one call (the rule by sorting is slow)."""
    tok, logp = TK.sample_tokens(logits, u, **kw)
    et, ep = _by_rule(logits[rows], u[rows], **{k: v[rows] if isinstance(v, torch.Tensor) else v for k, v in kw.items()})
    assert torch.equal(tok[rows], et)
    assert torch.allclose(logp[rows], ep, rtol=2.0 ** -22, atol=1e-6)


LONG = [dict(), dict(top_p=0.95), dict(top_p=0.9, temperature=0.3), dict(top_k=50, top_p=0.9), dict(top_k=60000), dict(min_p=0.05),
        dict(top_k=100000, top_p=0.99, temperature=2.0)]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("rule", LONG, ids=str)
@pytest.mark.parametrize("rows,vocab", [(148, 131072), (149, 262144), (160, 129001)])
def test_rows_as_long_as_they_come(rows, vocab, rule, dtype):
    """A block for each row, its threads adding more weights than 32 bits hold: logits close
    together, so that nearly all of them are of the largest's order, some masked, ties."""
    gen = torch.Generator("cuda").manual_seed(vocab)
    z = (0.5 * torch.randn(rows, vocab, generator=gen, device="cuda")).to(dtype)
    z[torch.rand(rows, vocab, generator=gen, device="cuda") < 0.02] = float("-inf")
    z[1] = 0.25
    z[2] *= 6
    _same_in([0, 1, 2, rows - 1], z, torch.rand(rows, 1, generator=gen, device="cuda"), **rule)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("rule", LONG, ids=str)
@pytest.mark.parametrize("rows,vocab", [(80, 20001), (40, 40000), (64, 131072), (20, 200003), (1, 262144), (3, 131073)])
def test_slices_of_every_size(rows, vocab, rule, dtype):
    """Clusters of 2 to 16 blocks whose slices are longer than 8192 candidates (rows enough to
    fill the GPU), and as long as they come in few rows."""
    gen = torch.Generator("cuda").manual_seed(vocab)
    z = (0.5 * torch.randn(rows, vocab + 1, generator=gen, device="cuda")).to(dtype)[:, 1:]
    z[torch.rand(rows, vocab, generator=gen, device="cuda") < 0.02] = float("-inf")
    z[rows // 2] *= 6
    _same_in(sorted({0, rows // 2, rows - 1}), z, torch.rand(rows, 1, generator=gen, device="cuda"), **rule)


@pytest.mark.parametrize("rows", [1, 150])
def test_order_across_the_bins(rows):
    """Logits a few representable numbers on both sides of every border of the histogram over
    exp(z): the limit by count falls between neighbours as their logits say, wherever it is."""
    border = torch.tensor([2.0 ** -o * (1 - j / 256) for o in range(36) for j in range(128)], dtype=torch.float64)
    at = border.log().float().cuda()
    bits = at.view(torch.int32)[:, None] + torch.arange(-6, 7, device="cuda", dtype=torch.int32)
    bits = torch.where((at == 0)[:, None], 0, bits)
    z = bits.view(torch.float32).flatten()
    gen = torch.Generator("cuda").manual_seed(6)
    z = z[torch.randperm(z.numel(), generator=gen, device="cuda")][None].expand(rows, -1)
    for k in torch.randint(1, z.shape[1], (12,), generator=gen, device="cuda").tolist() + [14, 15, 27]:
        u = torch.full((rows, 1), 1 - 2.0 ** -24, device="cuda")
        _same_in([0], z, u, top_k=k)
        _same_in([0], z, torch.rand(rows, 1, generator=gen, device="cuda"), top_k=k, top_p=0.7)
