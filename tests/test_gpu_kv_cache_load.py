"""Attention over the paged 8-bit KV cache under load: many sequences in a call (several to each thread that looks them over),
stretches of one sequence of more tiles than the tensor cores' sums are left unrounded for, and single tokens among chunks.
Bounds as for the small sizes (test_gpu_kv_cache.py)."""
import numpy as np
import pytest

from test_gpu_kv_cache import TYPES, check_attention, make, queries

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("name", TYPES)
@pytest.mark.parametrize("n, kv, group, hd, page, most", [(300, 2, 7, 64, 64, 1500), (700, 1, 1, 64, 16, 1100), (260, 2, 4, 128, 32, 1300),
                                                          (1030, 1, 3, 128, 128, 300)])
def test_many_sequences(qb, name, n, kv, group, hd, page, most):
    rng = np.random.default_rng(n)
    lens = rng.integers(0, most, n)
    lens[rng.integers(0, n, n // 4)] = rng.integers(0, 3, n // 4)  # runs of nearly empty ones
    lens[5] = most
    c = make(qb, lens.tolist(), kv, hd, page, seed=n)
    seqs = rng.permutation(n).tolist()
    check_attention(c, 0, queries(n, kv * group, hd, name), seqs, [1] * n, name=name)


@pytest.mark.parametrize("name", ["f32", "f16"])
@pytest.mark.parametrize("kv, hd, lens", [(8, 64, [140000]), (8, 128, [60011, 50000])])
def test_long_stretches_of_a_sequence(qb, name, kv, hd, lens):
    c = make(qb, lens, kv, hd, 128, seed=hd)
    check_attention(c, 0, queries(len(lens), kv, hd, name), list(range(len(lens))), [1] * len(lens), name=name)


@pytest.mark.parametrize("name", TYPES)
@pytest.mark.parametrize("kv, group, hd", [(4, 8, 128), (2, 7, 64)])
def test_single_tokens_among_chunks(qb, name, kv, group, hd):
    rng = np.random.default_rng(hd)
    lens = rng.integers(200, 2600, 20).tolist()
    news = [int(x) for x in rng.choice([0, 1, 1, 2, 17, 190], 20)]
    c = make(qb, lens, kv, hd, 32, seed=3)
    check_attention(c, 0, queries(sum(news), kv * group, hd, name), list(range(20)), news, name=name)
    check_attention(c, 0, queries(sum(news), kv * group, hd, name), list(range(20)), news, window=777, name=name)



def test_page_operations_of_the_largest_cache(qb):
    """2^20 pages and 8192 sequences: reserve, fork, free and compact, each over thousands of sequences in a call."""
    import torch
    n_pages, most = 1 << 20, 8192
    c = qb.PagedKV.empty(1, 1, 64, n_pages, most, 64, 16)
    rng = np.random.default_rng(0)
    lens = rng.integers(0, 900, most).astype(np.int32)
    half = most // 2
    lens[half:] = 0
    seqs = torch.randperm(most, device="cuda").to(torch.int32)
    c.reserve(seqs, torch.tensor(lens, device="cuda")[seqs.long()])
    c.check()
    used = int(((lens + 15) // 16).sum())
    assert c.lens.tolist() == lens.tolist() and int((c.refs > 0).sum()) == used and int((c.refs[:used] == 1).sum()) == used
    src = torch.arange(half, device="cuda", dtype=torch.int32)
    c.fork(src, src + half)
    c.check()
    own = int((lens[:half] % 16 != 0).sum())
    assert c.lens[half:].tolist() == lens[:half].tolist() and int((c.refs > 0).sum()) == used + own
    assert int(c.refs.sum()) == 2 * used
    c.free(src)
    c.check()
    assert int((c.refs > 0).sum()) == used and int((c.refs > 1).sum()) == 0
    c.compact()
    c.check()
    assert int((c.refs[:used] == 1).sum()) == used
    pages = c.table[half:][c.table[half:] >= 0]
    assert int((c.table[:half] >= 0).sum()) == 0 and torch.equal(pages.sort().values, torch.arange(used, device="cuda", dtype=torch.int32))
