"""RMS norm to 8-bit rows where a row's squares leave f32.  The bounds are those of test_gpu_decoder_rows.py."""
import math

import pytest

from test_gpu_decoder_rows import rows

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("name", ["f32", "bf16"])
@pytest.mark.parametrize("residual", [False, True])
@pytest.mark.parametrize("n", [32, 896, 4096, 8224, 32768])
@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf, 2e19, 3e38])
def test_a_row_whose_mean_square_is_no_number(qb, name, residual, n, bad):
    """One value that is not finite, or whose square is not: the whole row reads as NaN, the others as ever."""
    x = rows(3, n, name, seed=n)
    x[1, n // 2] = bad
    r = rows(3, n, name, seed=2) if residual else None
    h = x.double() + (0 if r is None else r.double())
    q, d = qb.rms_norm_q8(x, torch.ones(n, device="cuda"), residual=r)
    assert bool(d[1].isnan().all()) and not d[[0, 2]].isnan().any()
    got = qb.dequantize_q8(q, d, torch.float32).double()
    assert bool(got[1].isnan().all())
    y = (h / (h.square().mean(1, keepdim=True) + 1e-6).sqrt())[[0, 2]]
    assert bool((got[[0, 2]] - y).abs().le((0.5 + 3e-4) * d[[0, 2]].double().repeat_interleave(32, 1)).all())


@pytest.mark.parametrize("n", [32, 4096, 32768])
def test_the_largest_rows(qb, n):
    """A sum of squares just below f32's largest number, and just above it."""
    most = math.sqrt(2.0 ** 128 / n)
    sign = torch.where(torch.rand(2, n, generator=torch.Generator(device="cuda").manual_seed(n), device="cuda") < 0.5, -1.0, 1.0)
    x = sign * torch.tensor([[most * 0.999], [most * 1.001]], device="cuda")
    q, d = qb.rms_norm_q8(x, torch.ones(n, device="cuda"))
    assert torch.equal(q[0].float(), 127 * sign[0])
    assert bool(((d[0].double() - 1 / 127).abs() <= 32 * 2.0 ** -24 / 127).all()) and bool(d[1].isnan().all())
