"""The policy loss's definition where its terms are infinite."""
import torch

from surfb200.ops import rl as R


def test_a_kl_term_without_weight_takes_no_part():
    gen = torch.Generator().manual_seed(0)
    z = torch.randn(4, 6, generator=gen).requires_grad_()
    a = torch.tensor([0, 5, 2, 1])
    old, adv = torch.full((4,), -1.8), torch.tensor([1.0, -1.0, 0.5, 2.0])
    ref = torch.tensor([-1.0, 200.0, -float("inf"), -2.0])
    want, loss = R.policy_loss_reference(z, a, old, adv), R.policy_loss_reference(z, a, old, adv, ref_logp=ref)
    assert torch.equal(loss, want)
    assert torch.equal(torch.autograd.grad(loss, z)[0], torch.autograd.grad(want, z)[0])
