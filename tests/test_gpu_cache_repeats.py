"""Attention over the paged 8-bit KV cache, many times over: no wait of its kernels is missed (each gives up after seconds with an error
bit), and every call has the bits of the first."""
import time

import pytest

from test_gpu_kv_cache import TYPES, ints, make, queries

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("name", TYPES)
@pytest.mark.parametrize("hd, group, lens, news, window, calls", [
    (128, 4, [8191, 3000, 5111, 900, 7000, 1], [60, 509, 5, 100, 33, 1], 4096, 12000), (64, 7, [512], [512], 0, 20000),
    (64, 2, [70, 300, 200, 130], [17, 20, 200, 100], 0, 20000), (64, 7, [5000, 300, 20], [1, 1, 1], 0, 20000)])
def test_thousands_of_calls(qb, name, hd, group, lens, news, window, calls):
    if len(lens) == 6 and name != "f16":
        calls //= 3
    c = make(qb, lens, 2 if hd == 64 else 8, hd, 64, seed=70)
    q, starts = queries(sum(news), group * c.n_kv_heads, hd, name), [0]
    for m in news:
        starts.append(starts[-1] + m)
    args = (0, q, ints(range(len(lens))), ints(starts), max(news), max(lens))
    want = c.attention(*args, window=window)
    c.check()
    differ = torch.zeros((), dtype=torch.bool, device="cuda")
    began = time.monotonic()
    for i in range(calls):
        out = c.attention(*args, window=window)
        if i % 50 == 0:
            differ |= (out != want).any()
        if i % 1000 == 999:
            c.check()
            assert time.monotonic() - began < 10, "calls that take far too long"
    c.check()
    assert not differ
