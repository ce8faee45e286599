"""What the delta rule gives in 32 bits is made of 32-bit numbers with either type of token.

Final states, dA, ddt_bias and dstate are made of operands in three planes of bfloat16 (2^-24 of the number each),
bfloat16 tokens being exact in one. The bounds of 32-bit tokens therefore hold for bfloat16 ones too: 100 roundings of
2^-24 on the way through 25 chunks and the sums' own, 2^-24 sqrt(144) each: 7e-7 * 10, held to 1e-5, gradients (twice
as many) to 2e-5. With two planes (2^-16) anywhere on the way they would be held to 1e-4 and 2e-4.
"""
import pytest
import torch

from test_delta_gpu import BF, CASES, F32, INNER, MANY, NAMES, call, make, oracle, rel

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("case", CASES + MANY)
def test_32_bit_results_of_bfloat16_tokens(case):
    c = make(*case[:6], BF, case[6], case[7])
    _, final, want = oracle(c)
    r, d = call(c)
    assert rel(r.final, final) < INNER[F32]
    for n, x in zip(NAMES[5:], d[5:]):
        assert rel(x, want[n]) < 2 * INNER[F32], n


def test_reruns_of_long_rows_give_the_same_bits():
    """512 chunks one after the other, and many heads of many sequences."""
    for case in ((1, 8191, 8, 8, 128, 128, 0.0), (2, 4096, 16, 16, 64, 64, 0.0005), (256, 128, 8, 8, 64, 64, 0.02)):
        c = make(*case[:6], BF, case[6])
        c["A"] = c["A"] * 4 - 1
        (r, d), (r2, d2) = call(c), call(c)
        for x, y in zip((r.out, r.final, r.saved) + tuple(d), (r2.out, r2.final, r2.saved) + tuple(d2)):
            assert torch.equal(x, y)
