"""The memory core: its three ways to run agree with the float32 autograd statement, its
gradients too, and it learns to recall (CPU oracle; GPU kernels)."""
import numpy as np
import pytest
import torch

from surfb200.models import memory as M
from surfb200.ops import ssm, tokens as TK


def _small(device, seed=0):
    return M.MemoryNet(M.MemoryConfig(dim=32, rank=8, state=16), device, seed)


def test_recall_rows_follow_the_rule():
    t = M.RecallTask(5, longest=9, seed=1)
    x, r, want = t.rows(60)
    for e in range(5):
        cue = None
        for i in range(60):
            if r[e, i]:
                cue = int(np.argmax(x[e, i, :8]))
                assert x[e, i, :8].sum() == 1
            else:
                assert not x[e, i, :8].any()
            assert (want[e, i] >= 0) == bool(x[e, i, 8])
            if want[e, i] >= 0:
                assert want[e, i] == cue


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


def test_reference_gradients_by_differences():
    """Autograd of the definitions (float64) against differences: the oracles themselves."""
    gen = torch.Generator().manual_seed(0)
    r = lambda *s: torch.randn(*s, generator=gen, dtype=torch.float64)  # noqa: E731
    reset = torch.rand(2, 6, generator=gen) < 0.2
    n = torch.tensor([6, 4], dtype=torch.int32)
    p = [r(2, 6, 4), r(4, 3), r(4), r(2, 2, 4)]
    assert torch.autograd.gradcheck(
        lambda x, w, b, s: ssm.causal_conv_reference(x, w, b, state=s, reset=reset, lengths=n),
        [t.requires_grad_() for t in p])
    q = [r(2, 6, 4), r(2, 6, 4), -r(4, 3).abs(), r(2, 6, 2, 3), r(2, 6, 2, 3), r(4), r(2, 6, 4), r(4), r(2, 4, 3)]
    assert torch.autograd.gradcheck(
        lambda x, dt, A, B, C, D, z, b, s: ssm.selective_scan_reference(x, dt, A, B, C, D=D, z=z, dt_bias=b, state=s,
                                                                        reset=reset, lengths=n),
        [t.requires_grad_() for t in q])


def test_sampling_rule_on_small_rows():
    z = torch.tensor([[0.0, 2.0, 1.0, 2.0], [float("nan")] * 4, [-1.0, float("-inf"), -1.0, -5.0]])
    tok, logp = TK.sample_tokens_reference(z, torch.tensor([[0.0], [0.5], [0.99]]), top_k=2)
    assert tok[:, 0].tolist() == [1, -1, 2]
    assert logp[0, 0] == pytest.approx(-np.log(2)) and logp[1, 0] == float("-inf")
    # 0.9 of the weight is reached by the two largest; numbers spread over them as their shares
    p = torch.softmax(torch.tensor([0.0, 2.0, 1.0]), 0)
    u = torch.linspace(0, 0.999, 500)[:, None]
    tok, _ = TK.sample_tokens_reference(torch.tensor([[0.0, 2.0, 1.0]]).expand(500, 3), u, top_p=0.9)
    assert set(tok[:, 0].tolist()) == {1, 2}
    assert abs((tok == 1).float().mean() - p[1] / (p[1] + p[2])) < 0.01


def test_learns_on_cpu():
    r = M.train_recall(60, envs=32, length=16, cfg=M.MemoryConfig(dim=32, rank=8, answers=4), device="cpu", longest=5, act_steps=8)
    assert r["loss"][1] < 0.8 * r["loss"][0]


@pytest.mark.gpu
def test_sequence_and_gradients_match_the_reference():
    """bf16 operands: every projection rounds its inputs to 2^-9, five of them in a row and
    their errors independent: 2^-9 * sqrt(2 * 5) = 0.6% of the norm, held to 2%; gradients pass
    through twice as many, held to 4%."""
    cpu, net = _small("cpu"), _small("cuda")
    x, r, t = (torch.as_tensor(v) for v in M.RecallTask(6, longest=30).rows(50))
    params = cpu.autograd_params()
    for name in ("in.w", "x.w", "dt.w", "out.w"):                    # the operands the kernels read
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
    """Decision by decision through slots of a larger pool: the same logits up to the rounding
    of the windows and projections (each step rounds as the sequence does), states included."""
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
def test_learns_to_recall():
    r = M.train_recall(400)
    assert r["loss"][0] > 1.5 and r["loss"][1] < 1.0 and r["accuracy"] > 0.9, r


@pytest.mark.gpu
def test_reported_errors_are_raised(monkeypatch):
    """What a kernel reports while the core trains or answers ends the run, and is not left for
    whoever looks at the flag next."""
    from surfb200.ops import _lib
    from surfb200.ops import gemm as G
    G.check_error_flag("cuda")
    cfg = M.MemoryConfig(dim=32, rank=8)
    for iterations in (1, 25):
        G.error_flag("cuda").fill_(3)
        with monkeypatch.context() as m, pytest.raises(_lib.KernelError, match="epilogue wait"):
            if iterations == 25:                                     # raised before the answers
                m.setattr(M, "act", None)
            M.train_recall(iterations, envs=8, length=8, cfg=cfg, act_steps=1)
    G.check_error_flag("cuda")
    net = _small("cuda")
    state = M.MemoryState(net, 2)
    x = torch.zeros(2, 16, dtype=torch.bfloat16, device="cuda")
    M.act(net, x, state, torch.zeros(2, 1, device="cuda"), slots=torch.tensor([1, 2], dtype=torch.int32, device="cuda"))
    with pytest.raises(_lib.KernelError, match="state slot"):
        G.check_error_flag("cuda")
