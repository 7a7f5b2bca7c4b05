"""Windows of the attention over the paged 8-bit KV cache near the length's bound.  Bounds as in test_gpu_kv_cache.py."""
import pytest

from test_gpu_kv_cache import check_attention, ints, make, queries

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("n, kv, group, hd, length, window, m", [(64, 8, 4, 128, 1024, 1000, 1), (256, 2, 7, 64, 1000, 900, 1),
                                                                (1, 8, 4, 128, 4200, 4096, 4), (8, 8, 4, 128, 1000, 4096, 1),
                                                                (1, 8, 1, 64, 8000, 8192, 1), (64, 2, 4, 64, 1024, 1023, 4)])
def test_calls_near_the_window_are_served(qb, n, kv, group, hd, length, window, m):
    c = make(qb, [length - i % 3 for i in range(n)], kv, hd, 64, seed=n)
    check_attention(c, 0, queries(n * m, kv * group, hd, "bf16"), list(range(n)), [m] * n, name="bf16", window=window)


@pytest.mark.parametrize("window", [2 ** 31 - 1, 2 ** 31 - 5, 2 ** 30, 40 * 64, 40 * 64 - 1, 2000])
@pytest.mark.parametrize("lens, news", [([3, 0, 200, 2000], [10, 2, 5, 1]), ([3, 0, 200, 2000], [1, 1, 1, 1]), ([3, 0, 200, 300], [150, 70, 210, 301])])
def test_a_window_past_every_position_is_none(qb, lens, news, window):
    """Also for queries that sit far before position 0."""
    c = make(qb, lens, 2, 64, 64, seed=60, room=40 - max(-(-n // 64) for n in lens))
    assert c.table.shape[1] == 40
    q, starts = queries(sum(news), 4, 64, "f32"), [0]
    for m in news:
        starts.append(starts[-1] + m)
    for max_q in (max(news), 4 * max(news)):
        args = (0, q, ints(range(len(lens))), ints(starts), max_q, max(lens))
        want, wl = c.attention(*args, lse=True)
        out, lse = c.attention(*args, window=window, lse=True)
        c.check()
        if window >= 40 * 64:
            assert torch.equal(out, want) and torch.equal(lse, wl)
        else:  # the work may be dealt another way
            assert bool(((out - want).abs() <= 2.0 ** -16 * (1 + want.abs())).all())
    check_attention(c, 0, q, list(range(len(lens))), news, window=window)
