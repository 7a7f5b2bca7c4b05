"""Calls of the operators on torch tensors that are refused: counts past 32 bits."""
import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

MANY = 1 << 31


def test_more_tokens_than_a_call_takes(qb):
    """2^31 tokens are not 2^31 - 1: refused, nothing is written."""
    x, pos = torch.ones(MANY, 1, 2, dtype=torch.float16, device="cuda"), torch.ones(MANY, dtype=torch.int32, device="cuda")
    with pytest.raises(ValueError, match="2147483647"):
        qb.Rope(2)(x, None, pos, inplace=True)
    assert bool((x[:3] == 1).all()) and bool((x[-3:] == 1).all())
    del x
    one = torch.ones(1, 2, dtype=torch.float16, device="cuda").expand(MANY, 1, 2)
    with pytest.raises(ValueError, match="2147483647"):
        qb.Rope(2)(one, None, pos)
    del pos
    with pytest.raises(ValueError, match="2147483647"):
        qb.rms_norm_q8(torch.ones(32, device="cuda").expand(MANY, 32), torch.ones(32, device="cuda"))
