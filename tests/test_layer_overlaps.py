"""CPU checks of the calls around a decoder layer: rows that a call writes are refused where they share bytes with others that it
reads or writes.  Every call is one that is refused for something else where the rows are fine, so that nothing is launched."""
import random

import pytest

from test_kv_cache_abi import AT, INVALID, refused


def touched(at, stride, row, n):
    return {at + i * stride + j for i in range(n) for j in range(row)}


def rope(qb, q, qo, k, ko, n, heads=1, kv=1, dtype=1, hd=2):
    """(address, stride in elements) of each; no positions."""
    return qb.lib().qnt_rope(q[0], q[1], qo[0], qo[1], heads, k[0], k[1], ko[0], ko[1], kv, dtype, hd, hd, 0, AT, 1.0, None, n, None)


def test_rotated_heads_against_the_bytes_that_they_touch(qb):
    """Outputs and inputs with one stride anywhere around each other: refused exactly where they share a byte."""
    r, seen = random.Random(5), [0, 0]
    for _ in range(6000):
        n, heads, kv, hd = r.randint(1, 5), r.randint(1, 3), r.randint(1, 3), r.choice([2, 4])
        stride = max(heads, kv) * hd + r.randint(0, 12)
        rows = [max(heads, kv) * hd, heads * hd, kv * hd]
        q, k = AT, AT + 2 * r.randint(-80, 80)
        qo = q if r.random() < 0.5 else AT + 2 * r.randint(-80, 80)
        ko = k if r.random() < 0.5 else AT + 2 * r.randint(-80, 80)
        sets = {"q": touched(q, 2 * stride, 2 * rows[1], n), "qo": touched(qo, 2 * stride, 2 * rows[1], n),
                "k": touched(k, 2 * stride, 2 * rows[2], n), "ko": touched(ko, 2 * stride, 2 * rows[2], n)}
        bad = bool(sets["qo"] & sets["ko"] or sets["qo"] & sets["k"] or sets["q"] & sets["ko"] or
                   (q != qo and sets["q"] & sets["qo"]) or (k != ko and sets["k"] & sets["ko"]))
        refused(qb, rope(qb, (q, stride), (qo, stride), (k, stride), (ko, stride), n, heads, kv, 1, hd), INVALID,
                "overlap" if bad else "positions")
        seen[bad] += 1
    assert min(seen) > 1000


def test_rotated_heads_that_are_one_tensor(qb):
    refused(qb, rope(qb, (AT, 2), (AT, 2), (AT, 2), (AT, 2), 4), INVALID, "overlap")
    refused(qb, rope(qb, (AT, 2), (AT + 512, 2), (AT, 2), (AT + 1024, 2), 4), INVALID, "positions")  # (inputs may be the same)
    far = 2 ** 62  # (strides whose bytes pass 64 bits)
    refused(qb, rope(qb, (AT, far), (AT, far), (AT + 4, far), (AT + 4, far), 4), INVALID, "positions")
    refused(qb, rope(qb, (AT, far), (AT, far), (AT + 2, far), (AT + 2, far), 4), INVALID, "overlap")
    # a heads' count of 0 has no rows
    refused(qb, rope(qb, (AT, 2), (AT, 2), (None, 0), (None, 0), 4, kv=0), INVALID, "positions")


@pytest.mark.parametrize("dtype, rt, n, m, xs, r, rs", [
    (0, 0, 32, 1, 32, 4, 32), (0, 0, 32, 1, 32, -124, 32), (1, 1, 32, 2, 64, 62, 64), (1, 1, 32, 2, 64, -126, 64), (4, 4, 64, 3, 64, 128, 64),
    (4, 0, 64, 3, 64, 4, 64), (4, 0, 64, 3, 128, 128, 64), (0, 0, 32, 5, 40, 4 * 40 * 4, 40), (0, 0, 32, 5, 40, -4 * 40 * 4 + 124, 40)])
def test_residual_and_rows(qb, dtype, rt, n, m, xs, r, rs):
    size = 4 if dtype == 0 else 2
    rsize = 4 if rt == 0 else 2
    assert touched(AT, xs * size, n * size, m) & touched(AT + r, rs * rsize, n * rsize, m)
    rc = qb.lib().qnt_rms_norm_q8(AT, dtype, xs, AT + r, rt, rs, AT, 1e-6, m, n, 64 * AT, 65 * AT, None)
    refused(qb, rc, INVALID, "overlap")
