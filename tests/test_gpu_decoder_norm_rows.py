"""RMS norm to 8-bit rows where its kernels go on to another row, at exact halves, and where a row's squares leave f32.

The bounds are those of test_gpu_decoder_rows.py.  Halves: x of +-1 and eps = 0 make the mean square 1, its root 1 and y = weight; a
largest weight of 127 makes the scale 1, so that the codes are the weights, rounded."""
import math

import pytest

from test_gpu_decoder_rows import check_norm, rows

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("name", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("residual, pad, lead", [(None, 0, 0), ("same", 0, 0), ("f32", 0, 0), (None, 3, 1), ("same", 5, 3), ("f32", 1, 1)])
@pytest.mark.parametrize("m, n", [(4000, 288), (4500, 416), (700, 8224), (650, 16384), (400, 20000), (350, 32768)])
def test_more_rows_than_ctas(qb, name, residual, pad, lead, m, n):
    """Several warps and one chunk a thread; the 1024-thread kernels with two and four."""
    x = rows(m, n, name, seed=n, pad=pad, lead=lead)
    w = 1 + 0.3 * rows(1, n, "f32", seed=1, lead=lead)[0]
    r = None if residual is None else rows(m, n, name if residual == "same" else "f32", seed=2, pad=pad, lead=lead, std=3.0)
    check_norm(qb, x, w, 1e-6, r)


@pytest.mark.parametrize("name", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("m, n", [(1, 64), (3, 2048), (5, 8224), (1, 32768), (3000, 512)])
def test_halves_go_away_from_zero(qb, name, m, n):
    g = torch.Generator(device="cuda").manual_seed(n)
    x = torch.where(torch.rand(m, n, generator=g, device="cuda") < 0.5, -1.0, 1.0)
    v = torch.tensor([127, 0.5, -0.5, 1.5, -1.5, 2.5, 63.5, -126.5], device="cuda")
    w = torch.zeros(n, device="cuda").view(-1, 32)
    w[:, :8] = v
    w[:, 31] = 0.49999
    q, d = qb.rms_norm_q8(x.to({"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}[name]), w.view(-1), eps=0.0)
    want = torch.zeros_like(w)
    want[:, :8] = torch.tensor([127, 1, -1, 2, -2, 3, 64, -127], device="cuda")
    assert bool((d == 1).all())
    assert torch.equal(q.float(), (want.view(1, n) * x))


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
