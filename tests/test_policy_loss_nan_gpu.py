"""What the policy loss does with numbers that are not finite or far apart: NaN in what is known of a row shows in the
loss and in that row's gradient alone."""
import pytest
import torch

from surfb200.ops import rl as R
from test_policy_loss_gpu import BF, F32, call, make

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("v", [9, 300, 1001, 70000])
@pytest.mark.parametrize("name", ["old_logp", "advantages", "ref_logp", "weights"])
def test_nan_of_a_row_shows(name, v, dtype):
    c = make(7, v, dtype)
    c["answers"][4:6], c["logits"][4:6, :3] = 2, 0.5
    want = call(c, kl_coef=0.1, ent_coef=0.01)
    c[name] = c[name].clone()
    c[name][4] = float("nan")
    args = {k: None if t is None else t.double() for k, t in c.items() if k not in ("logits", "answers")}
    assert R.policy_loss_reference(c["logits"].double(), c["answers"], args.pop("old_logp"), args.pop("advantages"), **args, kl_coef=0.1,
                                   ent_coef=0.01).isnan()
    r = call(c, kl_coef=0.1, ent_coef=0.01)
    assert r.loss.isnan() and r.dlogits[4, :3].isnan().all()
    rest = torch.arange(7, device="cuda") != 4
    assert torch.equal(r.dlogits[rest], want.dlogits[rest])
    for x, y in zip((r.logp, r.kl, r.entropy), (want.logp, want.kl, want.entropy)):
        assert torch.equal(x[rest], y[rest])
    assert torch.equal(r.logp, want.logp) and torch.equal(r.entropy, want.entropy)


@pytest.mark.parametrize("v", [9, 1001])
def test_nan_of_a_row_without_advantage_shows_too(v):
    c = make(5, v, F32, masked=False)
    c["ref_logp"], c["advantages"][3] = None, 0.0
    c["old_logp"][3] = float("nan")
    r = call(c)
    assert r.loss.isnan() and r.dlogits[3].isnan().all() and torch.isfinite(r.dlogits[:3]).all()


@pytest.mark.parametrize("v", [9, 1001])
def test_nan_of_rows_that_count_nothing_stays_out(v):
    c = make(5, v, F32, masked=False)
    c["answers"][2] = -1
    want = call(c, kl_coef=0.1)
    for name in ("old_logp", "advantages", "ref_logp", "weights"):
        c[name] = c[name].clone()
        c[name][2] = float("nan")
    r = call(c, kl_coef=0.1)
    assert torch.isfinite(r.loss) and not r.dlogits[2].any()
    for x, y in zip(r, want):
        assert torch.equal(x, y)


@pytest.mark.parametrize("v", [9, 1001])
def test_a_kl_term_that_is_only_reported(v):
    """e^100 is infinite in 32 bits, and so is the KL term of a reference policy that gives an answer no probability."""
    c = make(5, v, F32, masked=False)
    plain = call(dict(c, ref_logp=None), ent_coef=0.01)
    for far in (100.0, -float("inf"), float("nan")):
        c["ref_logp"] = plain.logp + 0.3
        want = call(c, ent_coef=0.01)
        c["ref_logp"][1] = plain.logp[1] + far
        r = call(c, ent_coef=0.01)
        assert torch.equal(r.loss, plain.loss) and torch.equal(r.dlogits, plain.dlogits)
        assert not torch.isfinite(r.kl[1]) and torch.equal(r.kl[2:], want.kl[2:])
