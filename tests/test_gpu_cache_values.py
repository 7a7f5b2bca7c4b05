"""Attention over the paged 8-bit KV cache where values, scales or queries are unusual: scales of either sign and of very different
size, values and queries that are not finite.  Bounds as in test_gpu_kv_cache.py."""
import pytest

from test_gpu_kv_cache import SMALL, TYPES, check_attention, ints, make, queries

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("name", TYPES)
@pytest.mark.parametrize("hd", [64, 128])
def test_a_row_does_not_depend_on_values_it_cannot_see(qb, name, hd):
    """The last block's V, far larger than the others', is seen by the last queries alone: the rows before it keep their bits."""
    c = make(qb, [320, 1000], 2, hd, 64, seed=43)
    q, seqs, starts = queries(250, 4, hd, name), ints([0, 1]), ints([0, 200, 250])
    c.scales[..., 1, :, :] = torch.where(c.scales[..., 1, :, :] > 0, 2.0 ** -12, c.scales[..., 1, :, :])
    good = c.attention(0, q, seqs, starts, 200, 1000)
    for s, n in ((0, 320), (1, 1000)):
        c.scales[c.table[s, (n - 1) // 64].long(), 0, 1, :, (n - 1) % 64 // 16] = 2.0 ** 9
    out = c.attention(0, q, seqs, starts, 200, 1000)
    c.check()
    assert torch.equal(out[:184], good[:184]) and torch.equal(out[200:242], good[200:242])
    assert not torch.equal(out, good)


@pytest.mark.parametrize("name", TYPES)
@pytest.mark.parametrize("m", [1, 2, 60])
def test_large_values_of_keys_without_weight(qb, name, m):
    """The first block's V is 2^21 times the others', but its keys lie far behind in every score."""
    c = make(qb, [700], 1, 64, 64, seed=44)
    v = c.scales[:, 0, 1]
    v.copy_(torch.where(v > 0, 2.0 ** -12, v))
    p = c.table[0, 0].long()
    c.scales[p, 0, 1, 0, 0], c.scales[p, 0, 0, 0, 0] = 2.0 ** 9, 1.0
    c.codes[p, 0, 0, 0].view(4, 64, 16)[:, :16] = -127  # K of positions 0 .. 15
    check_attention(c, 0, queries(m, 8, 64, name).abs(), [0], [m], name=name)


@pytest.mark.parametrize("name", TYPES)
@pytest.mark.parametrize("m", [1, 30])
@pytest.mark.parametrize("sign", [1, -1])
def test_an_infinite_query_is_nan_whatever_its_scores(qb, name, m, sign):
    """All scores -inf (or +inf): the softmax of them is no number, as with scores of both signs."""
    c = make(qb, [300], 2, 64, 64, seed=45)
    c.codes[:, :, 0] = -5  # K
    q = queries(m, 6, 64, name).abs() + 0.1
    good = c.attention(0, q, ints([0]), ints([0, m]), m, 300)
    q2 = q.clone()
    q2[0, 2, 7] = sign * float("inf")
    out = c.attention(0, q2, ints([0]), ints([0, m]), m, 300)
    c.check()
    assert out[0, 2].isnan().all()
    keep = torch.ones(m, 6, dtype=torch.bool, device="cuda")
    keep[0, 2] = False
    assert torch.equal(out[keep], good[keep])


# lengths and queries of each sequence: single tokens in a CTA each, dealt out and joined by a warp and by a CTA a row; chunks whole and in stretches
SHAPES = {"few": ([200, 150, 90], [1, 1, 1]), "dealt": ([1500] * 20, [1] * 20), "long": ([9000], [1]), "chunk": ([200, 150, 300], [40, 150, 30]),
          "stretches": ([3000], [60])}


@pytest.mark.parametrize("name", TYPES)
@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("which, std", [("some", 1.5), ("some", 40.0), ("all", 1.5), ("all", 40.0)])
def test_scales_of_either_sign(qb, monkeypatch, shape, name, which, std):
    """value = code * scale whatever the scale's sign; also with scores far apart (results below 2^-126 may then read 0: where all
    keys but those with weights of 1e-60 have a 0 for V)."""
    monkeypatch.setitem(SMALL, name, SMALL[name] + 2.0 ** -126)
    lens, news = SHAPES[shape]
    c = make(qb, lens, 2, 64, 64, seed=41)
    g = torch.Generator(device="cuda").manual_seed(42)
    flip = torch.rand(c.scales.shape, generator=g, device="cuda") < (0.4 if which == "some" else 2.0)
    c.scales.copy_(torch.where(flip, -c.scales, c.scales))
    check_attention(c, 0, queries(sum(news), 6, 64, name, std=std), list(range(len(lens))), news, name=name)
    check_attention(c, 0, queries(sum(news), 6, 64, name, std=std), list(range(len(lens))), news, name=name, window=77)


@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf")])
@pytest.mark.parametrize("name", TYPES)
@pytest.mark.parametrize("shape", SHAPES)
def test_lse_does_not_depend_on_values(qb, shape, name, bad):
    """A V scale that is not finite: NaN for the queries that see it, whose lse (of scores alone) stays what it was."""
    lens, news = SHAPES[shape]
    c = make(qb, lens, 2, 64, 64, seed=40)
    q, starts = queries(sum(news), 6, 64, name), [0]
    for m in news:
        starts.append(starts[-1] + m)
    args = (0, q, ints(range(len(lens))), ints(starts), max(news), max(lens))
    good, gl = c.attention(*args, lse=True)
    at, pos = len(lens) - 1, lens[-1] - 20  # head 1 of the last sequence, the block of this position
    c.scales[c.table[at, pos // 64].long(), 0, 1, 1, pos % 64 // 16] = bad
    out, lse = c.attention(*args, lse=True)
    c.check()
    assert torch.equal(lse, gl)
    hit = torch.zeros(sum(news), 6, dtype=torch.bool, device="cuda")
    first = starts[-2] + max(0, pos // 16 * 16 - (lens[-1] - news[-1]))  # the first query that sees the block
    hit[first:, 3:] = True
    assert out[hit].isnan().all() and torch.equal(out[~hit], good[~hit])
