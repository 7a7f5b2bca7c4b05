"""The log sum of a long row whose tiles lie far below its largest logit: no rounding of the distance between them.

A row of 2^26 - 1 logits of -16 and one of 2^-20 (1 - 2^-7), whose distance is no f32 number: rounded to one it would be off by
9.4e-7, and so would 88% of the sum.  What is left: the exponential of the distance, 2^-22 and 2 roundings, and the tile with the
largest logit (12% of the sum, 12 roundings), together 0.88 (2.4e-7 + 1.2e-7) + 0.12 * 7.2e-7 < 4.1e-7."""
import math

import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("at", [0, 12345, (1 << 26) - 1])
def test_tiles_far_below_the_largest(qb, at):
    v, top = 1 << 26, 2.0 ** -20 * (1 - 2.0 ** -7)
    x = torch.full((1, 1, v), -16.0, device="cuda")
    x[0, 0, at] = top
    lse = math.log(math.exp(top) + (v - 1) * math.exp(-16.0))
    start = torch.tensor([[lse]], device="cuda")  # (so that the result is next to zero, where f32 is fine)
    scores, tokens, parents = qb.BeamSelector(1)(x, start)
    assert int(tokens) == at and int(parents) == 0
    assert abs(float(scores) - (float(start) + top - lse)) <= 4.1e-7
