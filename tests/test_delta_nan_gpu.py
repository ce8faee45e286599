"""NaN in the delta rule's tokens, gates and weights: it shows where the definition has it, in sequences and single
tokens alike, and reaches no other episode, row or head."""
import pytest
import torch

from surfb200.ops import delta as DR
from test_delta_gpu import BF, F32, INNER, call, make, oracle, rel

pytestmark = pytest.mark.gpu
BAD = 23


def spoiled(c, which, row=0):
    x = c["tokens"][which].clone()
    x[row, BAD] = float("nan")
    return dict(c, tokens=c["tokens"][:which] + (x,) + c["tokens"][which + 1:])


def steps(c):
    state, outs = c["state"].clone(), []
    for i in range(c["tokens"][0].shape[1]):
        reset = None if c["reset"] is None else c["reset"][:, i].contiguous()
        outs.append(DR.gated_delta_step(*(x[:, i] for x in c["tokens"]), c["A"], state, dt_bias=c["dt_bias"], reset=reset))
    return torch.stack(outs, 1), state


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("resets", [(), (21, 26, 28), (16,), (30,)])
@pytest.mark.parametrize("which", [1, 2, 3, 4])
@pytest.mark.parametrize("rows", [2, 151])
def test_a_token_that_is_nan_shows(rows, which, resets, dtype):
    """Of k, v, dt or b: its own output and all behind it in its episode, and the final state if that is the last."""
    c = make(rows, 50, 1, 2, 32, 32, dtype)
    if resets:
        c["reset"] = torch.zeros(rows, 50, dtype=torch.bool, device="cuda")
        c["reset"][:, list(resets)] = True
    clean, grads = call(c)
    c = spoiled(c, which)
    end = min([r for r in resets if r > BAD], default=50)
    begin = max([r for r in resets if r <= BAD], default=0)
    want, final, _ = oracle(c, grads=False)
    assert want[0, BAD:end].isnan().all()
    r, d = call(c)
    single, state = steps(c)
    for out, last in ((r.out, r.final), (single, state)):
        assert out[0, BAD:end].isnan().all()
        assert bool(last[0].isnan().all()) == (end == 50) and torch.isfinite(last[1:]).all()
        assert torch.isfinite(out[0, end:]).all() and torch.isfinite(out[0, :begin]).all()
    assert torch.isfinite(single[0, :BAD]).all()
    assert torch.equal(r.out[1:], clean.out[1:]) and torch.equal(r.final[1:], clean.final[1:])
    tol = torch.finfo(dtype).eps                       # episodes by themselves sum in another order
    assert rel(r.out[0, end:], clean.out[0, end:]) < INNER[dtype] + tol
    # its own gradients, and the weights' of which it is a part. Everything is linear in v: its own gradient has no v,
    # and a decay's has the values of the tokens before alone
    assert d.db[0, BAD].isnan().all() and d.ddt[0, BAD + (which == 2)].isnan().all()
    assert which == 2 or d.dv[0, BAD].isnan().all()
    assert d.dA.isnan().all() and d.ddt_bias.isnan().all()
    for x, y in zip(d[:5], grads[:5]):
        assert torch.isfinite(x[0, end:]).all() and torch.isfinite(x[0, :begin]).all() and torch.equal(x[1:], y[1:])


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("ragged", [False, True])
def test_a_bias_that_is_nan_shows_in_its_head(ragged, dtype):
    c = make(4, 40, 2, 2, 32, 48, dtype, reset=0.1, ragged=ragged)
    clean, grads = call(c)
    c["dt_bias"] = c["dt_bias"].clone()
    c["dt_bias"][1] = float("nan")
    check_head(c, clean, grads)


def check_head(c, clean, grads):
    """Head 1 of two, each with keys of its own: NaN in all its real tokens; head 0 to the bit as before."""
    r, d = call(c)
    n = c["lengths"]
    real = torch.ones(r.out.shape[:2], dtype=torch.bool, device="cuda") if n is None else \
        torch.arange(r.out.shape[1], device="cuda")[None] < n[:, None]
    assert r.out[:, :, 1][real].isnan().all() and not r.out[:, :, 1][~real].any()
    some = real.any(1)
    assert r.final[some, 1].isnan().all() and torch.equal(r.final[~some, 1], clean.final[~some, 1])
    assert torch.equal(r.out[:, :, 0], clean.out[:, :, 0]) and torch.equal(r.final[:, 0], clean.final[:, 0])
    assert d.dA[1].isnan() and d.ddt_bias[1].isnan() and d.dv[:, :, 1][real].isnan().all()
    for x, y in zip(d[:5], grads[:5]):
        assert torch.equal(x[:, :, 0], y[:, :, 0])
    assert torch.equal(d.dA[0], grads.dA[0]) and torch.equal(d.ddt_bias[0], grads.ddt_bias[0])
    assert torch.equal(d.dstate[:, 0], grads.dstate[:, 0])
    tokens = tuple(torch.nan_to_num(x[:, 0]) for x in c["tokens"])
    state = c["state"].clone()
    out = DR.gated_delta_step(*tokens, c["A"], state, dt_bias=c["dt_bias"])
    assert out[:, 1].isnan().all() and state[:, 1].isnan().all() and torch.isfinite(out[:, 0]).all() and torch.isfinite(state[:, 0]).all()


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("ragged", [False, True])
@pytest.mark.parametrize("rows", [4, 151])
def test_a_rate_that_is_nan_shows_in_its_head(rows, ragged, dtype):
    c = make(rows, 40, 2, 2, 32, 48, dtype, reset=0.1, ragged=ragged)
    clean, grads = call(c)
    c["A"] = c["A"].clone()
    c["A"][1] = float("nan")
    check_head(c, clean, grads)
