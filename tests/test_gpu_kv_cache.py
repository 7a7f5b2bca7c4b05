"""The paged 8-bit KV cache on the GPU: append, read, attention and the page operations against plain forms.

Attention is compared with the definition in 64 bits.  Bounds (u = 2^-24, all derived from the formula):
  a score is off by at most ds = (head_dim + 16) u scale sum_d |q_d k_d| (each product and sum rounded once, the query's
  fixed-point digits included), which changes a weight by a factor within exp(+-2 ds); the weights and sums themselves keep
  2^-17 (long sums in f32) for float32 queries and 2^-10 for 16-bit ones (weights may be held in 16 bits); a 16-bit
  result is rounded once more (a float16 one by up to 2^-25 where it is subnormal).  So |out - exact| <= (2 ds + w) sum_j
  p_j |v_j| + r |exact| (+ 2^-25), and |lse - exact| <= ds + 2^-19 (1 + |lse|).
Append is compared bit for bit with its f32 definition, and with the input within half a code.
"""
import numpy as np
import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
ROUND = {"f32": 2.0 ** -23, "f16": 2.0 ** -10, "bf16": 2.0 ** -7}
SMALL = {"f32": 0.0, "f16": 2.0 ** -25, "bf16": 0.0}
WEIGHT = {"f32": 2.0 ** -17, "f16": 2.0 ** -10, "bf16": 2.0 ** -10}


def ints(x):
    return torch.tensor(list(x), dtype=torch.int32, device="cuda")


def make(qb, lens, kv, hd, page, layers=1, spare=3, seed=0, n_pages=None, max_seqs=None, room=2):
    """A cache with sequences of these lengths in shuffled pages: random codes and scales, and NaN scales in every block
    that no sequence reaches (what is not in use must not matter)."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    need = [-(-n // page) for n in lens]
    n_pages = n_pages or sum(need) + spare
    c = qb.PagedKV.empty(layers, kv, hd, n_pages, max_seqs or max(1, len(lens)), max(need + [1]) + room, page)
    c.codes.copy_(torch.randint(-127, 128, c.codes.shape, generator=g, device="cuda", dtype=torch.int8))
    c.scales.fill_(float("nan"))
    order = torch.randperm(n_pages, generator=g, device="cuda").tolist()
    at = 0
    for s, n in enumerate(lens):
        for k in range(need[s]):
            p = order[at]
            at += 1
            c.table[s, k], c.refs[p] = p, 1
            blocks = -(-min(page, n - k * page) // 16)
            c.scales[p, ..., :blocks] = torch.exp(torch.randn(layers, 2, kv, blocks, generator=g, device="cuda") * 0.5) / 60
        c.lens[s] = n
    return c


def values(c, layer, seq, n=None):
    """(K, V) [len][kv][hd] of one sequence in f64, from the arrays."""
    pt, hd = c.page_tokens, c.head_dim
    n = int(c.lens[seq]) if n is None else n
    pages = c.table[seq, : -(-n // pt)].long()
    codes = c.codes[pages, layer].double()
    sc = c.scales[pages, layer].double().repeat_interleave(16, -1)  # [np][2][kv][pt]
    kv = c.n_kv_heads
    k = codes[:, 0].view(-1, kv, hd // 16, pt, 16).permute(0, 3, 1, 2, 4).reshape(-1, kv, hd)
    v = codes[:, 1].view(-1, kv, pt // 16, hd, 16).permute(0, 2, 4, 1, 3).reshape(-1, kv, hd)
    sc = sc.permute(1, 0, 3, 2).reshape(2, -1, kv, 1)
    return (k * sc[0])[:n], (v * sc[1])[:n]


def reference(c, layer, q, seqs, news, scale, window):
    """out, lse, and the bounds' parts: ds per row and sum_j p_j |v_j|."""
    outs, lses, dss, absv = [], [], [], []
    g, t0 = q.shape[1] // c.n_kv_heads, 0
    for s, m in zip(seqs, news):
        k, v = values(c, layer, s)
        n = k.shape[0]
        x = q[t0: t0 + m].double().view(m, c.n_kv_heads, g, c.head_dim)
        t0 += m
        pos, j = torch.arange(n - m, n, device="cuda"), torch.arange(n, device="cuda")
        seen = (j[None] <= pos[:, None]) & ((j[None] > pos[:, None] - window) if window else True)
        sc = (torch.einsum("mhgd,jhd->mhgj", x, k) * scale).masked_fill(~seen[:, None, None], -np.inf)
        mag = torch.einsum("mhgd,jhd->mhgj", x.abs(), k.abs()) * abs(scale)
        mag = mag.masked_fill(~seen[:, None, None], 0)
        dss.append((mag.amax(-1) if n else torch.zeros(m, c.n_kv_heads, g, dtype=torch.float64, device="cuda")).reshape(m, c.n_kv_heads * g)
                   * (c.head_dim + 16) * 2.0 ** -24)
        if n:
            p = torch.softmax(sc, -1).nan_to_num(0.0)  # a row that sees nothing: 0
            lses.append(torch.logsumexp(sc, -1).reshape(m, c.n_kv_heads * g))
        else:
            p = torch.zeros(m, c.n_kv_heads, g, 0, dtype=torch.float64, device="cuda")
            lses.append(torch.full((m, c.n_kv_heads * g), -np.inf, dtype=torch.float64, device="cuda"))
        outs.append(torch.einsum("mhgj,jhd->mhgd", p, v).reshape(m, c.n_kv_heads * g, c.head_dim))
        absv.append(torch.einsum("mhgj,jhd->mhgd", p, v.abs()).reshape(m, c.n_kv_heads * g, c.head_dim))
    return torch.cat(outs), torch.cat(lses), torch.cat(dss), torch.cat(absv)


def check_attention(c, layer, q, seqs, news, scale=None, window=0, name="f32", **more):
    starts = [0] + list(np.cumsum(news))
    max_len = max([int(c.lens[s]) for s in seqs] + [1])
    out, lse = c.attention(layer, q, ints(seqs), ints(starts), max(max(news), 1), max_len, scale=scale, window=window, lse=True,
                           **more)
    c.check()
    want, wl, ds, absv = reference(c, layer, q, seqs, news, c.head_dim ** -0.5 if scale is None else scale, window)
    tol = (2 * ds[..., None] + WEIGHT[name]) * absv + ROUND[name] * want.abs() + SMALL[name]
    bad = (out.double() - want).abs() > tol
    assert not bad.any() and not out.isnan().any(), (int(bad.sum()), float(((out.double() - want).abs() / (tol + 1e-300)).max()))
    none = wl == -np.inf
    assert torch.equal(lse == -np.inf, none) and not out[none].any()
    assert bool(((lse.double() - wl).abs()[~none] <= (ds + 2.0 ** -19 * (1 + wl.abs()))[~none]).all())
    return out


def queries(n_tok, heads, hd, name, seed=1, std=1.5):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn(n_tok, heads, hd, generator=g, device="cuda") * std).to(TYPES[name])


# ---------------------------------------------------------------- attention

@pytest.mark.parametrize("name", TYPES)
@pytest.mark.parametrize("kv, group, hd, page", [(2, 7, 64, 64), (1, 1, 128, 16), (3, 4, 128, 128), (2, 16, 64, 32), (1, 5, 64, 16),
                                                 (1, 8, 128, 64), (1, 40, 64, 64)])
def test_decode_lengths(qb, name, kv, group, hd, page):
    """One query per sequence, lengths about every boundary (blocks, pages, tiles) and none."""
    lens = [1, 2, 15, 16, 17, 31, 63, 64, 65, 127, 128, 129, 0, 255, 257, 300, 511, 513, 1000]
    c = make(qb, lens, kv, hd, page, seed=kv * group)
    seqs = list(np.random.default_rng(group).permutation(len(lens)))
    check_attention(c, 0, queries(len(lens), kv * group, hd, name), seqs, [1] * len(lens), name=name)


@pytest.mark.parametrize("name", TYPES)
@pytest.mark.parametrize("kv, group, hd, page, lens", [(2, 7, 64, 64, [4999]), (1, 2, 128, 32, [7777, 3, 4096]), (2, 1, 64, 16, [2500] * 5),
                                                       (1, 12, 64, 128, [9000, 0])])
def test_decode_long(qb, name, kv, group, hd, page, lens):
    """Few long sequences: their keys are split over many CTAs and joined."""
    c = make(qb, lens, kv, hd, page, seed=5)
    check_attention(c, 0, queries(len(lens), kv * group, hd, name), list(range(len(lens))), [1] * len(lens), name=name)


@pytest.mark.parametrize("name", TYPES)
@pytest.mark.parametrize("kv, group, hd, page, lens, news", [
    (2, 7, 64, 64, [512], [512]), (2, 7, 64, 64, [1, 2, 17, 130, 700], [1, 2, 17, 3, 129]), (1, 4, 128, 16, [300, 64, 1111], [1, 64, 200]),
    (1, 1, 64, 32, [513, 90], [257, 2]), (2, 3, 128, 128, [129, 128, 127], [5, 128, 127]), (1, 16, 64, 64, [1000, 40], [33, 40]),
    (1, 1, 128, 64, [2000], [15]), (1, 8, 64, 64, [3001], [2])])
def test_chunks(qb, name, kv, group, hd, page, lens, news):
    """Several queries per sequence, causal, from drafts of two tokens to whole prompts."""
    c = make(qb, lens, kv, hd, page, seed=9)
    check_attention(c, 0, queries(sum(news), kv * group, hd, name), list(range(len(lens))), news, name=name)


@pytest.mark.parametrize("window", [1, 5, 16, 100, 128, 4000])
@pytest.mark.parametrize("news", [[1, 1, 1, 1], [200, 1, 40, 3]])
def test_window(qb, window, news):
    c = make(qb, [700, 1, 129, 40], 2, 64, 64, seed=3)
    check_attention(c, 0, queries(sum(news), 6, 64, "f32"), [0, 1, 2, 3], news, window=window)


@pytest.mark.parametrize("name", ["f32", "f16"])
@pytest.mark.parametrize("kv, group", [(2, 7), (1, 1)])
def test_queries_before_the_first_position_see_nothing(qb, name, kv, group):
    """More queries than positions: the first ones sit before position 0; so does a query of an empty sequence."""
    c = make(qb, [3, 0, 5, 140], kv, 64, 16, seed=4)
    check_attention(c, 0, queries(10 + 2 + 5 + 150, kv * group, 64, name), [0, 1, 2, 3], [10, 2, 5, 150], name=name)
    check_attention(c, 0, queries(3, kv * group, 64, name), [1, 0, 2], [1, 1, 1], name=name)


def test_sequences_without_tokens_in_the_call(qb):
    c = make(qb, [100, 200, 300], 2, 64, 64, seed=6)
    check_attention(c, 0, queries(2, 14, 64, "f32"), [2, 0, 1], [1, 0, 1])
    check_attention(c, 0, queries(90, 14, 64, "f32"), [2, 0, 1], [0, 90, 0])


@pytest.mark.parametrize("name", TYPES)
@pytest.mark.parametrize("m", [1, 40])
def test_query_strides(qb, name, m):
    """Queries as a slice of wider rows that start at an odd element."""
    c = make(qb, [500, 70], 2, 64, 64, seed=8)
    wide = queries(2 * m, 30, 64, name).reshape(2 * m, -1)
    row = torch.empty(2 * m * 1921 + 1, dtype=wide.dtype, device="cuda")[1:].view(2 * m, 1921)
    row[:, :1920] = wide
    q = row[:, 3: 3 + 14 * 64].unflatten(1, (14, 64))
    check_attention(c, 0, q, [0, 1], [m, m], name=name)


@pytest.mark.parametrize("std, scale", [(0.0, None), (1e-20, None), (1e18, 1e-18), (30.0, None), (1.5, -0.3), (1.5, 0.0)])
@pytest.mark.parametrize("m", [1, 30])
def test_query_magnitudes(qb, std, scale, m):
    """All-zero, tiny, huge and very sharp scores, a negative and a zero scale."""
    c = make(qb, [333], 2, 64, 32, seed=11)
    check_attention(c, 0, queries(m, 14, 64, "f32", std=1.0) * std, [0], [m], scale=scale)


@pytest.mark.parametrize("m", [1, 30])
def test_one_large_value_among_many_small_ones(qb, m):
    """A key far ahead of the others, whose small weights still add up, and scales of very different size."""
    c = make(qb, [4000], 1, 64, 64, seed=12)
    c.codes[c.table[0, 0].long(), 0, 0] = 127
    p = c.table[0, :63].long()
    c.scales[p, 0, 1] = torch.nan_to_num(c.scales[p, 0, 1]) * torch.exp(torch.randn(63, 1, 4, device="cuda") * 6)
    check_attention(c, 0, queries(m, 4, 64, "f32").abs(), [0], [m])


@pytest.mark.parametrize("m", [1, 30])
def test_not_finite(qb, m):
    """A NaN or infinite value that a query sees makes its row NaN, and touches no other row, head or sequence."""
    c = make(qb, [200, 200, 150], 2, 64, 64, seed=13)
    q = queries(3 * m, 6, 64, "f32")
    starts = [0, m, 2 * m, 3 * m]
    good, gl = c.attention(0, q, ints([0, 1, 2]), ints(starts), m, 200, lse=True)
    q2 = q.clone()
    q2[m, 4, 17] = float("nan")   # sequence 1, head 4
    q2[m, 1, 3] = float("inf")
    c.scales[c.table[2, 1].long(), 0, 1, 1, 2] = float("nan")  # V of sequence 2, head 1, positions 96 .. 111
    out, _ = c.attention(0, q2, ints([0, 1, 2]), ints(starts), m, 200, lse=True)
    c.check()
    assert out[m, 4].isnan().all() and out[m, 1].isnan().all()
    assert out[2 * m:, 3:].isnan().all()
    keep = torch.ones(3 * m, 6, dtype=torch.bool, device="cuda")
    keep[m, 4] = keep[m, 1] = False
    keep[2 * m:, 3:] = False
    assert torch.equal(out[keep], good[keep])


def test_layers_and_shared_pages(qb):
    c = make(qb, [150, 90, 0], 2, 64, 32, layers=3, seed=14, max_seqs=4)
    c.fork(ints([0]), ints([2]))
    for layer in range(3):
        out = check_attention(c, layer, queries(3, 14, 64, "f32").expand(3, 14, 64), [0, 1, 2], [1, 1, 1])
        same = c.attention(layer, queries(1, 14, 64, "f32").expand(1, 14, 64).repeat(2, 1, 1), ints([0, 2]), ints([0, 1, 2]), 1, 150)
        assert torch.equal(same[0], same[1]) and out.shape == (3, 14, 64)


def test_pool_past_32_bits(qb):
    """Pages whose codes start past 2^31 and 2^32 bytes."""
    n_pages = (1 << 32) // (2 * 2 * 64 * 64) + 600
    c = qb.PagedKV.empty(1, 2, 64, n_pages, 2, 10, 64)
    g = torch.Generator(device="cuda").manual_seed(2)
    for s, pages in enumerate([[n_pages - 1, 3, n_pages // 2 + 7, n_pages - 300], [n_pages - 2, 140000 % n_pages]]):
        for k, p in enumerate(pages):
            c.table[s, k] = p
            c.codes[p] = torch.randint(-127, 128, c.codes.shape[1:], generator=g, device="cuda", dtype=torch.int8)
            c.scales[p] = 0.02
        c.lens[s] = 64 * len(pages) - 5
    check_attention(c, 0, queries(2, 14, 64, "f32"), [0, 1], [1, 1])
    check_attention(c, 0, queries(100, 14, 64, "f16"), [0, 1], [60, 40], name="f16")
    k, v = c.read(0, ints([0]), ints([0]), ints([0, 251]), 251)
    want = values(c, 0, 0)
    assert torch.equal(k.double(), want[0].float().double()) and torch.equal(v.double(), want[1].float().double())


@pytest.mark.parametrize("m", [1, 2, 77])
def test_same_bits_again_and_on_another_stream(qb, m):
    """No result depends on timing, on the stream, or on what the workspace held before."""
    c = make(qb, [6000, 100, 1300], 2, 64, 64, seed=15)
    q, seqs, starts = queries(3 * m, 14, 64, "f16"), ints([0, 1, 2]), ints([0, m, 2 * m, 3 * m])
    a = c.attention(0, q, seqs, starts, m, 6000)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        b = c.attention(0, q, seqs, starts, m, 6000)
    torch.cuda.current_stream().wait_stream(side)
    for ws in c._ws.values():
        ws.fill_(255)
    d = c.attention(0, q, seqs, starts, m, 6000)
    assert torch.equal(a, b) and torch.equal(a, d)


@pytest.mark.parametrize("m", [1, 9])
def test_a_longer_sequence_than_announced_is_read_whole(qb, m):
    c = make(qb, [3000, 10], 2, 64, 64, seed=16)
    q, seqs, starts = queries(2 * m, 14, 64, "f32"), ints([0, 1]), ints([0, m, 2 * m])
    want, wl, ds, absv = reference(c, 0, q, [0, 1], [m, m], 0.125, 0)
    out = c.attention(0, q, seqs, starts, m, 100, scale=0.125)
    c.check()
    assert bool(((out.double() - want).abs() <= (2 * ds[..., None] + WEIGHT["f32"]) * absv + ROUND["f32"] * want.abs()).all())


@pytest.mark.parametrize("m", [1, 20])
def test_bad_tables_are_reported(qb, m):
    """A sequence out of range, a missing page and a page past the pool are errors of check(), not faults."""
    c = make(qb, [300, 300], 2, 64, 64, seed=17)
    q, starts = queries(2 * m, 14, 64, "f32"), ints([0, m, 2 * m])
    good = c.attention(0, q, ints([0, 1]), starts, m, 300)
    for change in ("seq", "missing", "past"):
        seqs = ints([0, 7]) if change == "seq" else ints([0, 1])
        keep = c.table.clone()
        if change != "seq":
            c.table[1, 2] = -1 if change == "missing" else 10 ** 6
        out = c.attention(0, q, seqs, starts, m, 300)
        with pytest.raises(qb.QntError, match="out of range"):
            c.check()
        c.table.copy_(keep)
        assert torch.equal(out[:m], good[:m])
        c.check()


def test_graph_capture(qb):
    """A step (reserve, append, attention) captured once and replayed with new inputs."""
    c = make(qb, [100, 33], 2, 64, 64, seed=18, spare=8)
    q, k, v = (queries(2, h, 64, "f16", seed=s) for h, s in ((14, 1), (2, 2), (2, 3)))
    seqs, starts, one = ints([0, 1]), ints([0, 1, 2]), ints([1, 1])
    c.attention(0, q, seqs, starts, 1, 128)  # the workspace is made before the capture
    c.lens.copy_(ints([100, 33]))
    side, g = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        c.attention(0, q, seqs, starts, 1, 128)
    torch.cuda.synchronize()
    with torch.cuda.graph(g, stream=side):
        c.reserve(seqs, one)
        c.append(0, k, v, seqs, starts)
        out = c.attention(0, q, seqs, starts, 1, 128)
    for step in range(3):
        q.copy_(queries(2, 14, 64, "f16", seed=20 + step))
        k.copy_(queries(2, 2, 64, "f16", seed=30 + step))
        g.replay()
        torch.cuda.synchronize()
        assert c.lens.tolist() == [101 + step, 34 + step]
        want, wl, ds, absv = reference(c, 0, q, [0, 1], [1, 1], 0.125, 0)
        assert bool(((out.double() - want).abs() <= (2 * ds[..., None] + WEIGHT["f16"]) * absv + ROUND["f16"] * want.abs() + SMALL["f16"]).all())
    c.check()


# ---------------------------------------------------------------- append and read

def emulate(block_codes, old, x, kept):
    """The f32 definition of an append to one block: codes [16][hd] (the first `kept` live), old scale, x [m][hd] f32."""
    f = np.float32
    with np.errstate(all="ignore"):
        d = f(np.max(np.abs(x))) * (f(1) / f(127)) if x.size else f(0)
        d = f(d if not kept else (np.nan if np.isnan(old) or np.isnan(d) else max(f(old), d)))
        inv = f(1) / d if d > 0 else f(0)
        fine = d > 0 and np.isfinite(d) and np.isfinite(inv)
        out = np.zeros_like(block_codes)
        if kept:
            ratio = f(old) / d if fine else f(0)
            out[:kept] = block_codes[:kept] if d == old else np.rint(block_codes[:kept].astype(f) * ratio).astype(np.int8)
        if fine:
            out[kept: kept + len(x)] = np.clip(np.rint((x * inv).astype(f)), -127, 127).astype(np.int8)
    return out, d


def block_of(c, layer, kind, head, seq, b):
    """(codes [16][hd] int8, scale) of block b of a sequence."""
    pt, hd = c.page_tokens, c.head_dim
    page, t0 = int(c.table[seq, b * 16 // pt]), b * 16 % pt
    tile = c.codes[page, layer, kind, head].cpu().numpy()
    if kind == 0:
        codes = tile.reshape(hd // 16, pt, 16)[:, t0: t0 + 16].transpose(1, 0, 2).reshape(16, hd)
    else:
        codes = tile.reshape(pt // 16, hd, 16)[t0 // 16].T
    return codes.copy(), np.float32(c.scales[page, layer, kind, head, t0 // 16].item())


@pytest.mark.parametrize("name", TYPES)
@pytest.mark.parametrize("kv, hd, page", [(2, 64, 64), (3, 128, 16), (1, 64, 128), (5, 128, 32)])
def test_append_bit_for_bit(qb, name, kv, hd, page):
    """Single tokens, parts of blocks and whole prompts; rows as slices of a projection's output, aligned or not."""
    before, news = [0, 1, 15, 16, 40, 63, 100, 0, 33], [1, 1, 1, 1, 3, 2, 70, 150, 0]
    c = make(qb, before, kv, hd, page, layers=2, seed=21, spare=40, room=10)
    old = {(s, kind, h, b): block_of(c, 1, kind, h, s, b) for s, n in enumerate(before) for kind in (0, 1) for h in range(kv)
           for b in range(-(-n // 16))}
    other = c.codes[:, 0].clone()
    order = [3, 0, 8, 7, 1, 6, 5, 2, 4]
    seqs, starts = ints(order), [0] + list(np.cumsum([news[s] for s in order]))
    c.reserve(seqs, ints(news[s] for s in order))
    n_tok = starts[-1]
    for odd in (0, 1):  # the second time at an odd element: the same codes again
        g = torch.Generator(device="cuda").manual_seed(22)
        rows = torch.empty(n_tok * (2 * kv * hd + 3) + 1, dtype=TYPES[name], device="cuda")[odd:]
        rows = rows[: n_tok * (2 * kv * hd + 3)].view(n_tok, -1)
        x = (torch.randn(n_tok, 2, kv, hd, generator=g, device="cuda") * torch.exp(
            torch.randn(n_tok, 2, kv, 1, generator=g, device="cuda"))).to(TYPES[name])
        rows[:, : 2 * kv * hd] = x.reshape(n_tok, -1)
        k, v = (rows[:, i * kv * hd: (i + 1) * kv * hd].unflatten(1, (kv, hd)) for i in (0, 1))
        c.append(1, k, v, seqs, ints(starts))
        c.check()
        xs = x.float().cpu().numpy()
        for j, s in enumerate(order):
            p0, p1 = before[s], before[s] + news[s]
            for b in range(p0 // 16, -(-p1 // 16) if news[s] else 0):
                kept, end = max(p0 - 16 * b, 0), min(p1 - 16 * b, 16)
                for kind in (0, 1):
                    for h in range(kv):
                        was, scale = old.get((s, kind, h, b), (np.zeros((16, hd), np.int8), np.float32(0)))
                        part = xs[starts[j] + 16 * b + kept - p0: starts[j] + 16 * b + end - p0, kind, h]
                        want, d = emulate(was, scale, part, kept)
                        got, gd = block_of(c, 1, kind, h, s, b)
                        assert gd == d and np.array_equal(got, want), (s, b, kind, h, odd)
                        assert np.abs(got[kept:end] * np.float64(d) - part).max() <= d * (0.5 + 1e-4)
    assert torch.equal(c.codes[:, 0], other)  # the other layer is untouched
    for s, n in enumerate(before):  # and so is every block that the call did not reach
        for b in range(n // 16 if news[s] else -(-n // 16)):
            for kind in (0, 1):
                got, gd = block_of(c, 1, kind, 0, s, b)
                want, d = old[(s, kind, 0, b)]
                m = min(16, n - 16 * b)
                assert gd == d and np.array_equal(got[:m], want[:m])


def test_append_scale_grows_and_special_values(qb):
    c = qb.PagedKV.empty(1, 1, 64, 4, 2, 4, 16)
    one, starts = ints([0]), ints([0, 1])
    xs = np.zeros((8, 64), np.float32)
    xs[1], xs[2, 3], xs[3, 5], xs[4] = 0.01, -5.0, 100.0, 1e-42
    xs[6, 7] = np.inf
    codes, scale = np.zeros((16, 64), np.int8), np.float32(0)
    for i in range(8):
        c.reserve(one, ints([1]))
        row = torch.tensor(xs[i], device="cuda").view(1, 1, 64)
        c.append(0, row, row, one, starts)
        codes, scale = emulate(codes, scale, xs[i: i + 1], i)
        for kind in (0, 1):
            got, d = block_of(c, 0, kind, 0, 0, 0)
            assert (d == scale or (np.isnan(d) and np.isnan(scale))) and np.array_equal(got, codes), i
    k, v = c.read(0, one, ints([0]), ints([0, 8]), 8)
    assert k.isnan().all() and v.isnan().all()  # from the infinity on, the block reads as NaN
    # a block of values whose 1 / d is infinite holds zeros
    c.reserve(ints([1]), ints([2]))
    tiny = torch.full((2, 1, 64), 1e-40, device="cuda")
    c.append(0, tiny, tiny, ints([1]), ints([0, 2]))
    k, _ = c.read(0, ints([1]), ints([0]), ints([0, 2]), 2)
    assert not k.any()
    c.check()


@pytest.mark.parametrize("name", TYPES)
@pytest.mark.parametrize("kv, hd, page", [(2, 64, 64), (3, 128, 16), (1, 128, 128)])
def test_read(qb, name, kv, hd, page):
    lens = [1, 16, 33, 200, 0, 77]
    c = make(qb, lens, kv, hd, page, layers=2, seed=23)
    seqs, first, count = [3, 0, 2, 4, 5, 1], [5, 0, 16, 0, 76, 0], [190, 1, 17, 0, 1, 16]
    starts = [0] + list(np.cumsum(count))
    k, v = c.read(1, ints(seqs), ints(first), ints(starts), starts[-1], dtype=TYPES[name])
    c.check()
    for j, s in enumerate(seqs):
        wk, wv = values(c, 1, s)
        for got, want in ((k, wk), (v, wv)):
            w = want[first[j]: first[j] + count[j]].float().to(TYPES[name])  # one product rounded to f32, then to the type
            assert torch.equal(got[starts[j]: starts[j + 1]], w)
    c.read(1, ints([0]), ints([0]), ints([0, 2]), 2)  # past the sequence's end
    with pytest.raises(qb.QntError, match="out of range"):
        c.check()


def test_append_reports_what_does_not_fit(qb):
    c = make(qb, [5, 20], 1, 64, 16, seed=24)
    x = queries(9, 1, 64, "f32")
    for seqs, starts, bound in (([0], [0, 9], 9), ([9], [0, 1], 1), ([1], [0, 4], 2)):
        was = c.codes.clone()
        c.append(0, x, x, ints(seqs), ints(starts), bound)  # 9 new tokens of 5; no such sequence; more than announced
        with pytest.raises(qb.QntError, match="out of range"):
            c.check()
        assert torch.equal(was, c.codes)


# ---------------------------------------------------------------- pages

class Pool:
    """The page bookkeeping in plain Python."""

    def __init__(self, n_pages, max_seqs, page):
        self.refs, self.rows, self.lens, self.page = [0] * n_pages, [[] for _ in range(max_seqs)], [0] * max_seqs, page

    def take(self, n):
        free = [p for p, r in enumerate(self.refs) if r == 0]
        return None if len(free) < n else free[:n]

    def reserve(self, seqs, extra):
        want = [-(-(self.lens[s] + e) // self.page) - len(self.rows[s]) for s, e in zip(seqs, extra)]
        got = self.take(sum(want))
        if got is None:
            return False
        for s, e, w in zip(seqs, extra, want):
            for p in got[:w]:
                self.refs[p] = 1
            self.rows[s] += got[:w]
            got = got[w:]
            self.lens[s] += e
        return True

    def fork(self, src, dst):
        got = self.take(sum(self.lens[s] % self.page > 0 for s in src))
        if got is None:
            return None
        copies = []
        for s, d in zip(src, dst):
            self.rows[d], self.lens[d] = list(self.rows[s]), self.lens[s]
            if self.lens[s] % self.page:
                copies.append((self.rows[s][-1], got[0]))
                self.rows[d][-1] = got.pop(0)
            for p in self.rows[d]:
                self.refs[p] += 1
        return copies

    def free(self, seqs):
        for s in seqs:
            for p in self.rows[s]:
                self.refs[p] -= 1
            self.rows[s], self.lens[s] = [], 0

    def compact(self):
        n = sum(r > 0 for r in self.refs)
        moves = dict(zip([p for p in range(n, len(self.refs)) if self.refs[p]], [p for p in range(n) if not self.refs[p]]))
        for a, b in moves.items():
            self.refs[b], self.refs[a] = self.refs[a], 0
        self.rows = [[moves.get(p, p) for p in r] for r in self.rows]
        return list(moves.items())

    def equals(self, c):
        assert c.refs.tolist() == self.refs and c.lens.tolist() == self.lens
        t = c.table.tolist()
        for s, r in enumerate(self.rows):
            assert t[s][: len(r)] == r and all(x == -1 for x in t[s][len(r):]), s


@pytest.mark.parametrize("n_pages, max_seqs, page, layers, kv, hd", [(50, 12, 16, 2, 1, 64), (1000, 40, 32, 1, 2, 64), (64, 9, 64, 3, 1, 128),
                                                                     (33, 33, 128, 1, 1, 64), (40000, 300, 16, 1, 1, 64)])
def test_page_operations_follow_the_bookkeeping(qb, n_pages, max_seqs, page, layers, kv, hd):
    """Random reserves, forks, frees and compactions, the refused ones too: tables, counts and moved bytes as in Python."""
    rng = np.random.default_rng(n_pages)
    c, pool = qb.PagedKV.empty(layers, kv, hd, n_pages, max_seqs, 200, page), Pool(n_pages, max_seqs, page)
    g = torch.Generator(device="cuda").manual_seed(n_pages)
    c.codes.copy_(torch.randint(-127, 128, c.codes.shape, generator=g, device="cuda", dtype=torch.int8))
    c.scales.copy_(torch.rand(c.scales.shape, generator=g, device="cuda"))
    refused = 0
    for step in range(60):
        op = rng.choice(["reserve", "reserve", "fork", "free", "compact"])
        codes, scales, moved = c.codes.clone(), c.scales.clone(), []
        if op == "reserve":
            seqs = rng.permutation(max_seqs)[: rng.integers(1, max_seqs)]
            most = 4 * n_pages * page // max_seqs // 5
            extra = [int(min(rng.integers(0, most + 2), 200 * page - pool.lens[s])) for s in seqs]
            c.reserve(ints(seqs), ints(extra))
            ok = pool.reserve(list(seqs), extra)
        elif op == "fork":
            empty = [s for s in range(max_seqs) if not pool.lens[s]]
            rng.shuffle(empty)
            dst = empty[: rng.integers(0, max(1, min(10, len(empty))) + 1)]
            src = [int(s) for s in rng.integers(0, max_seqs, len(dst))]
            keep = [i for i, s in enumerate(src) if s not in dst]
            src, dst = [src[i] for i in keep], [dst[i] for i in keep]
            c.fork(ints(src), ints(dst))
            moved = pool.fork(src, dst)
            ok = moved is not None
        elif op == "free":
            seqs = rng.permutation(max_seqs)[: rng.integers(0, max(2, max_seqs // 2))]
            c.free(ints(seqs))
            pool.free(list(seqs))
            ok = True
        else:
            c.compact()
            moved, ok = pool.compact(), True
        if ok:
            c.check()
        else:
            refused += 1
            with pytest.raises(qb.QntError, match="no free pages"):
                c.check()
        pool.equals(c)
        if moved:
            a, b = (torch.tensor(x, device="cuda") for x in zip(*moved))
            codes[b], scales[b] = codes[a], scales[a]
        assert torch.equal(codes, c.codes) and torch.equal(scales, c.scales), op
    print("refused", refused)


def test_bad_lists_change_nothing(qb):
    c = make(qb, [40, 0, 70, 0], 1, 64, 16, seed=30, spare=30)
    was = [t.clone() for t in (c.refs, c.table, c.lens, c.codes)]
    bad = [lambda: c.reserve(ints([0, 0]), ints([1, 1])), lambda: c.reserve(ints([0, 4]), ints([1, 1])),
           lambda: c.reserve(ints([0, -1]), ints([1, 1])), lambda: c.reserve(ints([0, 2]), ints([1, -1])),
           lambda: c.reserve(ints([0]), ints([10 ** 6])), lambda: c.reserve(ints([0]), ints([2 ** 31 - 1])),
           lambda: c.fork(ints([0, 2]), ints([1, 1])), lambda: c.fork(ints([0]), ints([2])), lambda: c.fork(ints([0, 1]), ints([1, 3])),
           lambda: c.fork(ints([0]), ints([4])), lambda: c.fork(ints([-3]), ints([1])), lambda: c.fork(ints([0]), ints([0])),
           lambda: c.free(ints([0, 0])), lambda: c.free(ints([2, 4])), lambda: c.free(ints([-1])),
           lambda: c.copy_pages(ints([0]), ints([10 ** 6]))]
    for i, call in enumerate(bad):
        call()
        with pytest.raises(qb.QntError, match="out of range"):
            c.check()
        for t, w in zip((c.refs, c.table, c.lens, c.codes), was):
            assert torch.equal(t, w), i


def test_copy_pages(qb):
    c = make(qb, [500], 2, 64, 32, layers=2, seed=31, n_pages=40)
    c.scales.copy_(torch.rand(c.scales.shape, device="cuda"))
    codes, scales = c.codes.clone(), c.scales.clone()
    c.copy_pages(ints([3, 3, 8, 9]), ints([0, 39, 20, 9]))
    c.check()
    for a, b in ((3, 0), (3, 39), (8, 20)):
        codes[b], scales[b] = codes[a], scales[a]
    assert torch.equal(codes, c.codes) and torch.equal(scales, c.scales)


def test_refusals_of_the_python_class(qb):
    c = make(qb, [50], 2, 64, 16, seed=32)
    q, one, starts = queries(1, 14, 64, "f32"), ints([0]), ints([0, 1])
    with pytest.raises(TypeError):
        c.attention(0, q.double(), one, starts, 1, 50)
    with pytest.raises(TypeError):
        c.attention(0, q.cpu(), one, starts, 1, 50)
    with pytest.raises(TypeError):
        c.attention(0, q[:, :, :32], one, starts, 1, 50)
    with pytest.raises(TypeError):
        c.attention(0, q, one.long(), starts, 1, 50)
    with pytest.raises(ValueError):
        c.attention(0, q, one, one, 1, 50)
    with pytest.raises(qb.QntError, match="n_heads"):
        c.attention(0, q[:, :13], one, starts, 1, 50)
    with pytest.raises(qb.QntError, match="layer"):
        c.attention(1, q, one, starts, 1, 50)
    with pytest.raises(TypeError):
        c.append(0, q[:, :2], q[:, :2].half(), one, starts)
    with pytest.raises(TypeError):
        c.append(0, q[:, :3], q[:, :3], one, starts)
    with pytest.raises(ValueError):
        c.reserve(one, starts)
    with pytest.raises(TypeError):
        qb.PagedKV(c.codes.float(), c.scales, c.refs, c.table, c.lens)
    with pytest.raises(ValueError):
        qb.PagedKV(c.codes, c.scales[:5].contiguous(), c.refs, c.table, c.lens)
    with pytest.raises(qb.QntError, match="head_dim"):
        qb.PagedKV.empty(1, 1, 96, 4, 1, 1)
    c.check()
