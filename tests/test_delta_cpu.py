"""The oracles of the delta rule, group norm and policy loss by differences (float64), the rules that
they state on small cases, and the kernels' refusal of CPU tensors."""
import pytest
import torch

from surfb200.ops import _lib, delta as DR, norm as N, rl as R


def _r(gen, *s):
    return torch.randn(*s, generator=gen, dtype=torch.float64)


def test_delta_gradients_by_differences():
    gen = torch.Generator().manual_seed(0)
    reset = torch.rand(2, 5, generator=gen) < 0.3
    n = torch.tensor([5, 3], dtype=torch.int32)
    x = [_r(gen, 2, 5, 1, 4), _r(gen, 2, 5, 1, 4), _r(gen, 2, 5, 2, 3), _r(gen, 2, 5, 2), _r(gen, 2, 5, 2), -_r(gen, 2).abs(),
         _r(gen, 2), _r(gen, 2, 2, 3, 4)]
    assert torch.autograd.gradcheck(
        lambda q, k, v, dt, b, A, bias, s: DR.gated_delta_reference(q, k, v, dt, b, A, dt_bias=bias, state=s, reset=reset, lengths=n),
        [t.requires_grad_() for t in x])


def test_delta_recalls_what_was_written():
    """Orthogonal keys with beta = 1 and no decay: each key gives back the last value written under it."""
    eye = torch.eye(4, dtype=torch.float64)
    keys = eye[[0, 1, 2, 0, 1]].view(1, 5, 1, 4)
    v = torch.arange(10.0, dtype=torch.float64).view(1, 5, 1, 2)
    big = torch.full((1, 5, 1), 40.0, dtype=torch.float64)
    zero = torch.zeros(1, dtype=torch.float64)
    out, S = DR.gated_delta_reference(keys, keys, v, big * 0, big, zero, scale=1.0, normalize=False)
    torch.testing.assert_close(out, v)
    torch.testing.assert_close(S[0, 0] @ eye[0], v[0, 3, 0])
    torch.testing.assert_close(S[0, 0] @ eye[2], v[0, 2, 0])


@pytest.mark.parametrize("activation", ["none", "silu"])
def test_norm_gradients_by_differences(activation):
    gen = torch.Generator().manual_seed(1)
    x = [_r(gen, 2, 3, 6), _r(gen, 6), _r(gen, 6)]
    assert torch.autograd.gradcheck(lambda x, w, b: N.group_norm_reference(x, 2, w, b, activation=activation),
                                    [t.requires_grad_() for t in x])


def test_norm_is_torch_group_norm():
    gen = torch.Generator().manual_seed(2)
    x, w, b = _r(gen, 3, 5, 7, 12), _r(gen, 12), _r(gen, 12)
    want = torch.nn.functional.group_norm(x.permute(0, 3, 1, 2), 4, w, b).permute(0, 2, 3, 1)
    torch.testing.assert_close(N.group_norm_reference(x, 4, w, b), want)


def test_policy_loss_gradients_by_differences():
    gen = torch.Generator().manual_seed(3)
    z = _r(gen, 5, 7)
    a = torch.tensor([0, 3, -1, 6, 2])
    lp = torch.log_softmax(z / 0.7, 1).gather(1, a.clamp(min=0)[:, None])[:, 0]
    old, ref, adv = lp - torch.tensor([0.1, -0.1, 0.0, 0.5, -0.5]), lp + 0.3, torch.tensor([1.0, -1.0, 1.0, 1.0, -1.0], dtype=torch.float64)
    f = lambda z: R.policy_loss_reference(z, a, old, adv, ref_logp=ref, kl_coef=0.2, ent_coef=0.1, temperature=0.7)  # noqa: E731
    assert torch.autograd.gradcheck(f, [z.requires_grad_()])
    # rows 3 and 4 are past their border: only the KL and the entropy move them
    g = torch.autograd.grad(R.policy_loss_reference(z, a, old, adv, temperature=0.7), z)[0]
    assert g[:2].any(1).all() and not g[2:].any()


def test_policy_loss_matches_the_heads_loss():
    """One head, no reference policy: the clipped term of the trainer's loss on the same numbers."""
    gen = torch.Generator().manual_seed(4)
    z = _r(gen, 6, 4)
    a = torch.randint(0, 4, (6,), generator=gen)
    old, adv = _r(gen, 6) * 0.1 - 1.4, _r(gen, 6)
    lp = torch.log_softmax(z, 1).gather(1, a[:, None])[:, 0]
    ratio = torch.exp(lp - old)
    want = torch.max(-adv * ratio, -adv * ratio.clamp(0.8, 1.2)).mean()
    torch.testing.assert_close(R.policy_loss_reference(z, a, old, adv), want)


def test_kernels_refuse_cpu_tensors():
    z = torch.zeros(2, 3)
    with pytest.raises(_lib.KernelError):
        R.policy_loss(z, torch.zeros(2, dtype=torch.int32), z[:, 0], z[:, 0])
    with pytest.raises(_lib.KernelError):
        N.group_norm(z, 1)
    with pytest.raises(_lib.KernelError):
        DR.gated_delta(*(torch.zeros(1, 2, 1, 4),) * 3, torch.zeros(1, 2, 1), torch.zeros(1, 2, 1), torch.zeros(1))
