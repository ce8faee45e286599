"""The delta rule's calls without tokens or rows: states pass through, gradients of the weights are zero."""
import pytest
import torch

from surfb200.ops import delta as DR
from test_delta_gpu import BF, F32, call, make

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("rows", [0, 3, 160])
@pytest.mark.parametrize("g,h,nk,nv", [(1, 1, 8, 8), (1, 2, 8, 8), (2, 6, 24, 40), (1, 1, 16, 65), (2, 2, 128, 128), (1, 3, 64, 100)])
def test_no_tokens(g, h, nk, nv, rows, dtype):
    """One key head for each value head or for several, values of one block or of two."""
    c = make(rows, 0, g, h, nk, nv, dtype)
    c["reset"] = torch.zeros(rows, 0, dtype=torch.bool, device="cuda")
    r, d = call(c)
    assert torch.equal(r.final, c["state"]) and torch.equal(d.dstate, c["dfinal"])
    for x, t in zip((r.out,) + d[:5], (c["tokens"][2],) + c["tokens"]):
        assert x.shape == t.shape and x.dtype == t.dtype
    assert not d.dA.any() and not d.ddt_bias.any()
    c["dfinal"] = None
    assert not call(c)[1].dstate.any()


@pytest.mark.parametrize("dtype", [BF, F32])
def test_rows_of_no_tokens(dtype):
    """Lengths of zero in every row: outputs and gradients of the tokens are zeros, the tokens are not read."""
    c = make(5, 33, 1, 2, 32, 100, dtype)
    c["lengths"] = torch.zeros(5, dtype=torch.int32, device="cuda")
    c["tokens"] = tuple(torch.full_like(x, float("nan")) for x in c["tokens"])
    c["dout"] = torch.full_like(c["dout"], float("nan"))
    r, d = call(c)
    assert torch.equal(r.final, c["state"]) and torch.equal(d.dstate, c["dfinal"])
    for x in (r.out,) + tuple(d[:7]):
        assert not x.any()


def test_no_rows_of_single_tokens():
    c = make(2, 1, 1, 2, 16, 16, BF)
    before = c["state"].clone()
    out = DR.gated_delta_step(*(x[:0, 0] for x in c["tokens"]), c["A"], c["state"])
    assert out.shape == (0, 2, 16) and torch.equal(c["state"], before)
