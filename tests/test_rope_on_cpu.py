"""Rotary positions of CPU tensors: refused as wrong arguments before any device work."""
import pytest

torch = pytest.importorskip("torch")


def test_tensors_of_the_cpu(qb):
    rope = qb.Rope(8, device="cpu")
    q, pos = torch.ones(2, 3, 8), torch.arange(2, dtype=torch.int32)
    for inplace in (False, True):
        with pytest.raises(TypeError, match="CUDA"):
            rope(q, None, pos, inplace=inplace)
        with pytest.raises(TypeError, match="CUDA"):
            rope(q, q.clone(), pos, inplace=inplace)
    assert bool((q == 1).all())
