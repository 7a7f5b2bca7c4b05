"""PagedKV.reorder: the sequences' contents, the page table and the reference counts against a plain model of them."""
import numpy as np
import pytest

from test_gpu_kv_cache import ints, make, queries, values

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu


def beams(qb, groups, width, lens, prompts, kv=2, hd=64, page=16, layers=2, spare=None, seed=0, room=2):
    """A cache of groups of `width` sequences; a group's share the full pages of their prompt."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    rng = np.random.default_rng(seed)
    n = groups * width
    each = [lens[i // width] if np.ndim(lens[0]) == 0 else lens[i // width][i % width] for i in range(n)]
    need = [-(-x // page) for x in each]
    shared = [min(prompts[i // width] // page, min(each[i // width * width: (i // width + 1) * width]) // page) for i in range(n)]
    pages = sum(shared[::width]) + sum(need) - sum(shared) + (n if spare is None else spare)
    c = qb.PagedKV.empty(layers, kv, hd, pages, n + 3, max(need + [1]) + room, page)
    c.codes.copy_(torch.randint(-127, 128, c.codes.shape, generator=g, device="cuda", dtype=torch.int8))
    c.scales.copy_(torch.exp(torch.randn(c.scales.shape, generator=g, device="cuda") * 0.5) / 60)
    order, at = rng.permutation(pages).tolist(), 0
    seqs = rng.permutation(n + 3)[:n].tolist()
    table, refs, lens_ = c.table.cpu().numpy(), np.zeros(pages, np.int32), np.zeros(n + 3, np.int32)
    for j in range(groups):
        common = order[at: at + shared[j * width]]
        at += len(common)
        for i in range(j * width, (j + 1) * width):
            own = order[at: at + need[i] - len(common)]
            at += len(own)
            row = common + own
            table[seqs[i], : len(row)] = row
            refs[row] += 1
            lens_[seqs[i]] = each[i]
    c.table.copy_(torch.from_numpy(table))
    c.refs.copy_(torch.from_numpy(refs))
    c.lens.copy_(torch.from_numpy(lens_))
    return c, seqs


def model(c, seqs, parents, group):
    """Table, refs and lens after the call, and the copies (from, to, blocks)."""
    pt = c.page_tokens
    table, refs, lens = c.table.cpu().numpy().copy(), c.refs.cpu().numpy().copy(), c.lens.cpu().numpy().copy()
    rows, old_lens = {s: table[s].copy() for s in seqs}, lens.copy()
    place = [i - i % group + p for i, p in enumerate(parents)]
    heir = {}
    for i, j in enumerate(place):
        heir.setdefault(j, i)
    for i, j in enumerate(place):
        if i == j:
            heir[j] = i
    for s in seqs:
        used = rows[s][rows[s] >= 0]
        refs[used] -= 1
    fresh = []
    for i, j in enumerate(place):
        row, n = rows[seqs[j]].copy(), old_lens[seqs[j]]
        if n % pt and heir[j] != i:
            fresh.append((i, n // pt, row[n // pt], -(-(n % pt) // 16)))
            row[n // pt] = -1
        refs[row[row >= 0]] += 1
        table[seqs[i]], lens[seqs[i]] = row, n
    free = np.flatnonzero(refs == 0)
    if len(free) < len(fresh):
        return None
    copies = []
    for (i, k, src, blocks), dst in zip(fresh, free):
        table[seqs[i], k] = dst
        refs[dst] = 1
        copies.append((int(src), int(dst), blocks))
    return table, refs, lens, copies


def check(c, seqs, parents, group=None, **more):
    group_ = len(seqs) if group is None else group
    want = model(c, seqs, parents, group_)
    codes, scales = c.codes.clone(), c.scales.clone()
    before = [[values(c, l, s) for l in range(c.n_layers)] for s in seqs]
    c.reorder(ints(seqs), ints(parents), group, **more)
    c.check()
    table, refs, lens, copies = want
    assert np.array_equal(c.table.cpu().numpy(), table)
    assert np.array_equal(c.refs.cpu().numpy(), refs)
    assert np.array_equal(c.lens.cpu().numpy(), lens)
    # the copies' filled blocks, and nothing else anywhere
    pt, hd = c.page_tokens, c.head_dim
    for src, dst, blocks in copies:
        k = codes.view(*codes.shape[:4], -1)
        a, b = k[src, :, 0].view(c.n_layers, c.n_kv_heads, hd // 16, pt, 16), k[dst, :, 0].view(c.n_layers, c.n_kv_heads, hd // 16, pt, 16)
        b[:, :, :, : blocks * 16] = a[:, :, :, : blocks * 16]
        codes[dst, :, 1, :, : blocks * 16 * hd] = codes[src, :, 1, :, : blocks * 16 * hd]
        scales[dst, ..., :blocks] = scales[src, ..., :blocks]
    assert torch.equal(c.codes, codes) and torch.equal(c.scales, scales)
    for i, p in enumerate(parents):  # every sequence reads what its parent did
        j = i - i % group_ + p
        for l in range(c.n_layers):
            for a, b in zip(values(c, l, seqs[i]), before[j][l]):
                assert torch.equal(a, b)


@pytest.mark.parametrize("page", [16, 32, 64, 128])
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("groups, width, lo, hi", [(1, 1, 5, 5), (1, 4, 100, 100), (3, 4, 1, 300), (20, 8, 30, 700), (2, 60, 90, 130)])
def test_reorder(qb, page, hd, groups, width, lo, hi):
    rng = np.random.default_rng(page + hd + groups)
    lens = rng.integers(lo, hi + 1, groups).tolist()
    c, seqs = beams(qb, groups, width, lens, [n // 2 for n in lens], hd=hd, page=page, layers=2 if hd == 64 else 1, seed=groups)
    for step in range(3):
        check(c, seqs, rng.integers(0, width, groups * width).tolist(), width)


@pytest.mark.parametrize("parents", [[0, 1, 2, 3, 4, 5], [5, 4, 3, 2, 1, 0], [1, 2, 3, 4, 5, 0], [0] * 6, [5] * 6, [1, 1, 3, 3, 5, 5],
                                     [2, 2, 2, 0, 0, 1]], ids=str)
@pytest.mark.parametrize("lens", [[40, 33, 48, 1, 0, 64], [48] * 6, [0] * 6, [17] * 6], ids=str)
def test_who_continues_whom(qb, parents, lens):
    """Identities, turns, one parent for all; lengths that differ, that end with a page, that are zero."""
    c, seqs = beams(qb, 1, 6, [lens], [0], seed=3)
    check(c, seqs, parents)
    check(c, seqs, parents)


def test_pages_freed_by_the_call_are_there_for_its_copies(qb):
    """A full pool: the dropped beams' pages are the copies'; with one page too few, nothing changes."""
    c, seqs = beams(qb, 1, 4, [[40, 40, 40, 40]], [32], spare=0, seed=4)
    check(c, seqs, [2, 2, 2, 2])
    check(c, seqs, [3, 3, 1, 0])
    c, seqs = beams(qb, 1, 3, [[48, 48, 40]], [48], spare=0, seed=5)  # two beams without a page of their own
    check(c, seqs, [2, 2, 2])
    c2, seqs2 = beams(qb, 1, 3, [[32, 32, 40]], [32], spare=0, seed=6)
    assert model(c2, seqs2, [2, 2, 2], 3) is None
    before = [t.clone() for t in (c2.codes, c2.scales, c2.refs, c2.table, c2.lens)]
    c2.reorder(ints(seqs2), ints([2, 2, 2]))
    with pytest.raises(qb.QntError, match="no free pages"):
        c2.check()
    assert all(torch.equal(a, b) for a, b in zip(before, (c2.codes, c2.scales, c2.refs, c2.table, c2.lens)))
    c2.check()
    check(c2, seqs2, [2, 0, 1])  # (needs none)


@pytest.mark.parametrize("seqs, parents", [([0, 1, 1], [0, 0, 0]), ([0, 1, 99], [0, 0, 0]), ([0, -1, 2], [0, 0, 0]), ([0, 1, 2], [0, 3, 0]),
                                           ([0, 1, 2], [0, -1, 0])])
def test_refused_lists_change_nothing(qb, seqs, parents):
    c, _ = beams(qb, 1, 3, [[40, 50, 60]], [0], seed=7)
    before = [t.clone() for t in (c.codes, c.scales, c.refs, c.table, c.lens)]
    c.reorder(ints(seqs), ints(parents))
    with pytest.raises(qb.QntError, match="out of range"):
        c.check()
    assert all(torch.equal(a, b) for a, b in zip(before, (c.codes, c.scales, c.refs, c.table, c.lens)))


def test_a_page_that_the_table_has_wrong(qb):
    """A part-filled page whose number is not the pool's: reported, nothing changes."""
    c, seqs = beams(qb, 1, 3, [[40, 40, 40]], [0], seed=8)
    c.table[seqs[1], 2] = 10 ** 6
    before = [t.clone() for t in (c.codes, c.scales, c.refs, c.table, c.lens)]
    c.reorder(ints(seqs), ints([1, 1, 1]))
    with pytest.raises(qb.QntError, match="out of range"):
        c.check()
    assert all(torch.equal(a, b) for a, b in zip(before, (c.codes, c.scales, c.refs, c.table, c.lens)))


@pytest.mark.parametrize("pages", [300000, 1 << 20])
def test_large_pool_and_many_sequences(qb, pages):
    """Shared memory of the plan past 48 KB, and at its most; a search of 1020 groups of 8."""
    c, seqs = beams(qb, 1020, 8, [20] * 1020, [16] * 1020, layers=1, kv=1, page=16, spare=pages - 1020 * 9, seed=9)
    assert c.refs.numel() == pages
    rng = np.random.default_rng(9)
    want = model(c, seqs, p := rng.integers(0, 8, 8160).tolist(), 8)
    c.reorder(ints(seqs), ints(p), 8)
    c.check()
    for a, b in zip((c.table, c.refs, c.lens), want):
        assert np.array_equal(a.cpu().numpy(), b)


def test_beams_go_on_apart(qb):
    """After a reordering children of one parent append different tokens: each reads its own, attention sees them."""
    c, seqs = beams(qb, 2, 3, [30, 45], [16, 32], layers=1, seed=10)
    s, starts = ints(seqs), ints(range(7))
    kept = []
    for step, parents in enumerate([[0, 0, 0, 2, 2, 1], [1, 0, 1, 2, 1, 0], [2, 2, 2, 0, 1, 2]]):
        before = [values(c, 0, q)[0] for q in seqs]
        c.reorder(s, ints(parents), 3)
        c.reserve(s, ints([1] * 6))
        k, v = queries(6, 2, 64, "f32", seed=20 + step), queries(6, 2, 64, "f32", seed=40 + step)
        c.append(0, k, v, s, starts, 1)
        out = c.attention(0, queries(6, 4, 64, "f32", seed=60 + step), s, starts, 1, 64)
        c.check()
        for i, q in enumerate(seqs):
            got, was = values(c, 0, q)[0], before[i // 3 * 3 + parents[i]]
            assert got.shape[0] == was.shape[0] + 1
            block = was.shape[0] // 16 * 16  # (an append rounds its block's earlier codes again)
            assert torch.equal(got[:block], was[:block])
            d = c.scales[c.table[q, was.shape[0] // 16], 0, 0, :, 0].double()
            assert bool(((got[-1] - k[i].double()).abs() <= 0.51 * d[:, None]).all())
        assert out.isfinite().all()


def test_streams_and_graphs(qb):
    c, seqs = beams(qb, 4, 4, [40, 33, 100, 64], [32] * 4, seed=11)
    start = [t.clone() for t in (c.codes, c.scales, c.refs, c.table, c.lens)]
    s, p = ints(seqs), ints([3, 3, 1, 0] * 4)
    side = torch.cuda.Stream()

    def reset():
        for t, b in zip((c.codes, c.scales, c.refs, c.table, c.lens), start):
            t.copy_(b)
        torch.cuda.synchronize()

    c.reorder(s, p, 4)
    torch.cuda.synchronize()
    want = [t.clone() for t in (c.codes, c.scales, c.refs, c.table, c.lens)]
    for stream in (side, side.cuda_stream, 0):
        reset()
        c.reorder(s, p, 4, stream=stream)
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(want, (c.codes, c.scales, c.refs, c.table, c.lens)))
    reset()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=side):
        c.reorder(s, p, 4)
    p.copy_(ints([0, 0, 2, 2] * 4))
    torch.cuda.synchronize()
    expect = model(c, seqs, [0, 0, 2, 2] * 4, 4)
    g.replay()
    torch.cuda.synchronize()
    for a, b in zip((c.table, c.refs, c.lens), expect):
        assert np.array_equal(a.cpu().numpy(), b)
    c.check()


def test_lists_are_checked(qb):
    c, seqs = beams(qb, 1, 4, [20], [0], seed=12)
    with pytest.raises(ValueError):
        c.reorder(ints(seqs), ints([0, 0]))
    with pytest.raises(TypeError):
        c.reorder(ints(seqs).long(), ints([0] * 4))
    with pytest.raises(qb.QntError, match="whole groups"):
        c.reorder(ints(seqs), ints([0] * 4), 3)
    with pytest.raises(qb.QntError, match="whole groups"):
        c.reorder(ints(seqs), ints([0] * 4), 0)
    c.reorder(ints([]), ints([]))
    c.check()
