"""Sequences that a call cannot have, between good ones: reported by check(), and the good ones' results are right."""
import numpy as np
import pytest

from test_gpu_kv_cache import ROUND, SMALL, TYPES, WEIGHT, ints, make, queries, reference

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("name", TYPES)
@pytest.mark.parametrize("n, most, m", [(300, 1500, 1), (40, 6000, 1), (300, 900, 1), (60, 1500, 2), (12, 900, 40)])
@pytest.mark.parametrize("kind", ["unknown", "just past", "negative", "too many rows", "rows past the end", "all of them"])
def test_refused_sequences_between_good_ones(qb, name, n, most, m, kind):
    rng = np.random.default_rng(n)
    lens = rng.integers(most // 2, most, n).tolist()
    c = make(qb, lens, 2, 64, 64, seed=n)
    seqs, news = rng.permutation(n).tolist(), [m] * n
    bad = sorted(rng.choice(n, max(3, n // 5), replace=False).tolist() + [n // 2, n // 2 + 1])  # two that follow one another among them
    if kind == "all of them":
        bad = list(range(n))
    if kind == "rows past the end":
        bad = [n - 2, n - 1]
    wrong = list(seqs)
    for j in bad:
        if kind == "too many rows":
            news[j] = m + 1
        elif kind != "rows past the end":
            wrong[j] = {"unknown": 10 ** 6, "negative": -5}.get(kind, n)
    starts = [0] + list(np.cumsum(news))
    n_tok = starts[-1]
    if kind == "rows past the end":
        n_tok = starts[n - 2]
    q = queries(n_tok, 6, 64, name)
    out = c.attention(0, q, ints(wrong), ints(starts), m, most)
    if kind == "rows past the end":
        c.check()  # (rows that the call does not have: nothing to compute)
    else:
        with pytest.raises(qb.QntError, match="out of range"):
            c.check()
    for j in [j for j in range(n) if j not in bad][:: max(1, n // 25)]:
        part = slice(starts[j], starts[j + 1])
        want, _, ds, absv = reference(c, 0, q[part], [seqs[j]], [news[j]], 0.125, 0)
        tol = (2 * ds[..., None] + WEIGHT[name]) * absv + ROUND[name] * want.abs() + SMALL[name]
        assert bool(((out[part].double() - want).abs() <= tol).all()), j
