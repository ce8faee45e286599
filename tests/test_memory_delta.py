"""The memory core on the delta rule, and answers trained by the policy loss: the ways to run it agree with the
float32 autograd statement, its gradients too (CPU oracle; GPU kernels)."""
import pytest
import torch

from surfb200.models import memory as M
from surfb200.ops import rl as R, tokens as TK


def _small(device, seed=0):
    return M.MemoryNet(M.MemoryConfig(dim=64, core="delta", heads=4, keys=16), device, seed)


def test_reference_in_pieces_equals_whole():
    net = _small("cpu")
    x, r, _ = (torch.as_tensor(v) for v in M.RecallTask(3, longest=7).rows(20))
    s = M.MemoryState(net, 3)
    whole, _, _ = net.forward_reference(x, s, r)
    parts = []
    for lo, hi in ((0, 1), (1, 8), (8, 20)):
        y, s.conv, s.scan = net.forward_reference(x[:, lo:hi], s, r[:, lo:hi])
        parts.append(y)
    torch.testing.assert_close(torch.cat(parts, 1), whole, rtol=1e-5, atol=1e-5)


def test_refused_configurations():
    for bad in (dict(core="lstm"), dict(core="delta", heads=3), dict(core="delta", heads=4, dim=1024), dict(core="delta", keys=12),
                dict(core="delta", keys=136)):
        with pytest.raises(ValueError):
            M.MemoryNet(M.MemoryConfig(**bad))
    with pytest.raises(ValueError, match="objective"):
        M.train_recall(1, objective="luck", device="cpu")


@pytest.mark.parametrize("core", ["scan", "delta"])
@pytest.mark.parametrize("objective", ["answers", "policy"])
def test_runs_on_cpu(core, objective):
    cfg = M.MemoryConfig(dim=32, rank=8, answers=4, core=core, heads=4, keys=8)
    r = M.train_recall(3, envs=8, length=12, cfg=cfg, device="cpu", longest=5, act_steps=2, objective=objective)
    assert all(torch.isfinite(torch.tensor(r["loss"]))) and 0.0 <= r["accuracy"] <= 1.0


@pytest.mark.gpu
@pytest.mark.parametrize("core", ["scan", "delta"])
@pytest.mark.parametrize("objective", ["answers", "policy"])
def test_runs_on_gpu(core, objective):
    cfg = M.MemoryConfig(dim=64, rank=8, core=core, heads=4, keys=16)
    r = M.train_recall(26, envs=16, length=40, cfg=cfg, act_steps=3, objective=objective)
    assert all(torch.isfinite(torch.tensor(r["loss"]))) and 0.0 <= r["accuracy"] <= 1.0


@pytest.mark.gpu
def test_sequence_and_gradients_match_the_reference():
    """bf16 operands: the features' projections, the convolution, the heads' outputs and the norm's round to
    2^-8 at most (2^-9 on average), six in a row with errors of their own: 2^-8 sqrt(6) = 1% of the norm, held
    to 2%; gradients pass through twice as many, held to 4%. Keys of 16 numbers add the correction's
    own: an error of a key is one of what it reads and writes."""
    cpu, net = _small("cpu"), _small("cuda")
    x, r, _ = (torch.as_tensor(v) for v in M.RecallTask(6, longest=30).rows(50))
    params = cpu.autograd_params()
    for name in ("in.w", "gate.w", "out.w"):                         # the operands the kernels read
        params[name].data.copy_(params[name].data.bfloat16().float())
    s = M.MemoryState(cpu, 6)
    xb = x.bfloat16()
    want, _, _ = cpu.forward_reference(xb.float(), s, r, params)
    d = torch.randn(want.shape, generator=torch.Generator().manual_seed(1)).bfloat16()
    (want * d.float()).sum().backward()
    sg = M.MemoryState(net, 6)
    got, cache = M.forward_sequence(net, xb.cuda(), sg, r.cuda())
    rel = lambda a, b: float((a.float().cpu() - b).norm() / b.norm())  # noqa: E731
    assert rel(got, want.detach()) < 0.02
    M.backward(net, cache, d.cuda())
    for name, _ in net.specs:
        assert rel(net.g(name), params[name].grad) < 0.04, name


@pytest.mark.gpu
def test_steps_follow_the_sequence():
    net = _small("cuda")
    x, r, _ = (torch.as_tensor(v).cuda() for v in M.RecallTask(5, longest=12).rows(33))
    seq = M.MemoryState(net, 5)
    want, _ = M.forward_sequence(net, x.bfloat16(), seq, r, train=False)
    pool = M.MemoryState(net, 9)
    slots = torch.tensor([8, 0, 3, 4, 6], dtype=torch.int32, device="cuda")
    for i in range(33):
        got = M.step(net, x[:, i].bfloat16(), pool, reset=r[:, i].contiguous(), slots=slots)
        assert float((got - want[:, i]).norm() / want[:, i].norm()) < 1e-2
    at = slots.long()
    assert torch.equal(pool.conv[at], seq.conv)
    assert float((pool.scan[at] - seq.scan).norm() / seq.scan.norm()) < 1e-2


@pytest.mark.gpu
def test_policy_gradient_matches_the_reference():
    """A batch of rows answered by sample_tokens and one policy-loss gradient of the whole core, kernels against autograd."""
    cpu, net = _small("cpu"), _small("cuda")
    x, r, t = (torch.as_tensor(v) for v in M.RecallTask(16, longest=10).rows(40))
    sg = M.MemoryState(net, 16)
    logits, cache = M.forward_sequence(net, x.bfloat16().cuda(), sg, r.cuda())
    u = torch.rand(t.numel(), 1, generator=torch.Generator().manual_seed(2))
    a = M._Answered(logits, t.cuda(), net.cfg, u.cuda(), TK.sample_tokens)
    d = torch.zeros_like(logits)
    R.policy_loss(logits.view(-1, 64)[:, :8], a.answers, a.logp, a.advantages, out=d.view(-1, 64)[:, :8], **a.options())
    M.backward(net, cache, d.bfloat16())
    params = cpu.autograd_params()
    for name in ("in.w", "gate.w", "out.w"):
        params[name].data.copy_(params[name].data.bfloat16().float())
    want, _, _ = cpu.forward_reference(x.bfloat16().float(), M.MemoryState(cpu, 16), r, params)
    opts = {k: v.cpu() if isinstance(v, torch.Tensor) else v for k, v in a.options().items()}
    R.policy_loss_reference(want.view(-1, 64)[:, :8], a.answers.cpu(), a.logp.cpu(), a.advantages.cpu(), **opts).backward()
    for name, _ in net.specs:
        g = params[name].grad
        # as of the sequence's gradients; ratios near 1 amplify nothing
        assert float((net.g(name).cpu() - g).norm() / g.norm()) < 0.05, name


def test_no_epochs_are_refused():
    with pytest.raises(ValueError, match="epochs"):
        M.train_recall(1, device="cpu", objective="policy", epochs=0)
