"""Outputs whose rows share memory with one another are refused before anything is launched."""
import pytest
import torch

from surfb200.ops import delta as DR, norm as N, ssm as S, tokens as TK

pytestmark = pytest.mark.gpu


def test_refusals():
    r = lambda *s: torch.randn(*s, device="cuda")  # noqa: E731
    buf = torch.zeros(4096, device="cuda")
    tokens = (r(2, 5, 2, 16), r(2, 5, 2, 16), r(2, 5, 2, 16), r(2, 5, 2), r(2, 5, 2), -torch.ones(2, device="cuda"))
    one = tuple(x[:, 0] for x in tokens[:5]) + tokens[5:]
    x = r(3, 6, 32)
    calls = {
        "sequence": lambda: DR.gated_delta(*tokens, out=buf.as_strided((2, 5, 2, 16), (160, 16, 16, 1))),
        "single": lambda: DR.gated_delta_step(*one, r(2, 2, 16, 16), out=buf.as_strided((2, 2, 16), (8, 16, 1))),
        "norm": lambda: N.group_norm(x, 4, out=buf.as_strided((3, 6, 32), (192, 20, 1))),
        "in place": lambda: N.group_norm(buf.as_strided((3, 6, 32), (192, 20, 1)), 4, out=buf.as_strided((3, 6, 32), (192, 20, 1))),
        "convolution": lambda: S.causal_conv(x, r(32, 4), out=buf.as_strided((3, 6, 32), (192, 20, 1))),
    }
    for name, call in calls.items():
        with pytest.raises(ValueError, match="out has elements that share memory"):
            call()
            pytest.fail(name)
    assert not buf.any()
    # rows apart are taken, wherever they lie
    want = N.group_norm(x, 4).out
    got = N.group_norm(x, 4, out=buf.as_strided((3, 6, 32), (32, 100, 1))).out
    assert torch.equal(got, want)
    tok, _ = TK.sample_tokens(x[0], torch.rand(6, 1, device="cuda"))
    assert tok.shape == (6, 1)
