"""The selection of a beam search's next step on the GPU, against its definition in 64 bits: the tokens and beams have to be the
definition's; a score is within 2.7e-6 plus its rounding, 2^-24 of itself.  A row's log sum, whose relative error is the mean of
its terms' and of the roundings behind them: an exponential 2^-22 = 2.4e-7, its argument in units of log 2, 32 at most where it
counts, half a step ln 2 * 2^-20 = 6.6e-7 and log2 e as f32 21 * 1.4e-8 = 3.0e-7; 12 roundings in a tile's sum 7.2e-7; a tile's weight
2.4e-7; 8 roundings in the row's 4.8e-7.  Together 2.64e-6."""
import math

import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
INF = math.inf


def expected(logits, scores, k, ended=None, end_id=-1):
    x, s = logits.double(), scores.double()
    g, b, v = x.shape
    s = torch.where(s.isfinite(), s, -INF)
    c = s[..., None] + (x - torch.logsumexp(x, -1, keepdim=True))
    c = torch.where(c.isnan(), -INF, c)
    if ended is not None:
        only = torch.full_like(c, -INF)
        only[..., end_id] = s
        c = torch.where(ended.bool()[..., None], only, c)
    best, at = c.flatten(1).sort(dim=-1, descending=True, stable=True)
    return best[:, :k], (at % v)[:, :k].int(), (at // v)[:, :k].int()


def check(qb, logits, scores, k, ended=None, end_id=-1, select=None):
    scores_, tokens, parents = (select or qb.BeamSelector(k, end_id=end_id))(logits, scores, ended)
    want = expected(logits, scores, k, ended, end_id)
    assert scores_.shape == tokens.shape == parents.shape == (logits.shape[0], k)
    assert torch.equal(parents, want[2]) and torch.equal(tokens, want[1])
    w = want[0]
    none = w == -INF
    assert torch.equal(scores_ == -INF, none)
    assert bool(((scores_.double() - w).abs()[~none] <= (2.7e-6 + 2.0 ** -24 * w.abs())[~none]).all())


def make(g, b, v, name, seed=0, std=3.0):
    r = torch.Generator(device="cuda").manual_seed(seed)
    return ((torch.randn(g, b, v, generator=r, device="cuda") * std).to(TYPES[name]),
            -torch.rand(g, b, generator=r, device="cuda") * 5)


@pytest.mark.parametrize("name", TYPES)
@pytest.mark.parametrize("g, b, v, k", [(1, 1, 1, 1), (1, 4, 151665, 4), (3, 1, 5000, 64), (2, 3, 7, 21), (2, 3, 7, 5), (5, 2, 2049, 33),
                                        (1, 16, 8193, 32), (7, 5, 50257, 10), (64, 4, 8000, 8), (2, 64, 3001, 64), (300, 1, 16385, 1),
                                        (1, 1, 70000, 31), (1, 1000, 33, 40)])
def test_select(qb, name, g, b, v, k):
    check(qb, *make(g, b, v, name, seed=v), k)


@pytest.mark.parametrize("name", TYPES)
@pytest.mark.parametrize("lead, pad", [(1, 0), (3, 5), (7, 1), (0, 7), (5, 8)])
@pytest.mark.parametrize("v", [5, 9000])
def test_rows_at_any_address(qb, name, lead, pad, v):
    """Rows that start anywhere within 16 bytes; what lies around them is not looked at."""
    r = torch.Generator(device="cuda").manual_seed(lead)
    buf = torch.full((6 * (v + pad) + lead + 9,), INF, device="cuda", dtype=TYPES[name])
    x = buf[lead: lead + 6 * (v + pad)].view(2, 3, v + pad)[..., :v]
    x.copy_(torch.randn(2, 3, v, generator=r, device="cuda") * 2)
    check(qb, x, -torch.rand(2, 3, generator=r, device="cuda"), 9)


@pytest.mark.parametrize("name", TYPES)
@pytest.mark.parametrize("k", [1, 8, 40, 64])
@pytest.mark.parametrize("kind", ["all equal", "few values", "two values", "zeros of both signs", "rising", "falling", "one stretch"])
def test_equal_and_ordered_logits(qb, name, k, kind):
    """Ties go to the lowest place, whatever else; orders for which a threshold lets most candidates pass."""
    g, b, v = 2, 3, 20000
    r = torch.Generator(device="cuda").manual_seed(k)
    x = {"all equal": lambda: torch.full((g, b, v), 1.5, device="cuda"),
         "few values": lambda: torch.randint(0, 5, (g, b, v), generator=r, device="cuda").float(),
         "two values": lambda: (torch.rand(g, b, v, generator=r, device="cuda") < 0.01).float() * 4,
         "zeros of both signs": lambda: torch.where(torch.rand(g, b, v, generator=r, device="cuda") < 0.5, 0.0, -0.0),
         "rising": lambda: (torch.arange(v, device="cuda") * 5e-4).expand(g, b, v).contiguous(),
         "falling": lambda: (torch.arange(v, device="cuda") * -5e-4).expand(g, b, v).contiguous(),
         "one stretch": lambda: torch.where(torch.arange(v, device="cuda") // 300 == 7, 10.0, 0.0).expand(g, b, v) +
         torch.randn(g, b, v, generator=r, device="cuda") * 0.1}[kind]()
    check(qb, x.to(TYPES[name]), -torch.rand(g, b, generator=r, device="cuda") * 3, k)


@pytest.mark.parametrize("name", TYPES)
def test_beams_that_are_alike(qb, name):
    """Equal candidates of several beams: the lowest beam first."""
    x, s = make(3, 1, 6000, name, seed=1)
    check(qb, x.expand(3, 4, 6000).contiguous(), s.expand(3, 4).contiguous(), 20)
    few = torch.randint(0, 3, (1, 1, 6000), device="cuda").to(TYPES[name]).expand(2, 5, 6000).contiguous()
    check(qb, few, torch.zeros(2, 5, device="cuda"), 50)


@pytest.mark.parametrize("name", TYPES)
@pytest.mark.parametrize("step", [2.0 ** -29, -(2.0 ** -29), 2.0 ** -24, -(2.0 ** -22)])
@pytest.mark.parametrize("v", [3000, 151936])
def test_candidates_next_to_each_other(qb, name, step, v):
    """The same logits in another order, and a score that differs by almost nothing: the sums' roundings must not decide."""
    r = torch.Generator(device="cuda").manual_seed(v)
    x, _ = make(4, 1, v, name, seed=2)
    order = torch.stack([torch.randperm(v, generator=r, device="cuda") for _ in range(4)])[:, None]
    both = torch.cat([x, x.gather(2, order)], 1)
    s = torch.full((4, 2), -(2.0 ** -6), device="cuda")
    s[:, 1] += step
    assert bool((s[:, 0] != s[:, 1]).all())
    check(qb, both, s, 16)


@pytest.mark.parametrize("name", TYPES)
@pytest.mark.parametrize("k", [1, 2, 3, 4, 5, 7, 8])
@pytest.mark.parametrize("copies, beams", [(1, 3), (3, 2), (3, 4), (40, 3)])
@pytest.mark.parametrize("v, apart", [(700, True), (6000, True), (6000, False)])
def test_equal_logits_next_to_another_beam(qb, name, k, copies, beams, v, apart):
    """The last kept candidates have equals in their own beam, and another beam's lie closer than the sums' roundings: whichever beam
    is ahead in truth is kept.  Equals across tiles, or next to each other."""
    r = torch.Generator(device="cuda").manual_seed(100 * copies + k)
    x = torch.randn(64, 1, v, generator=r, device="cuda") * 2
    top = torch.randperm(v, generator=r, device="cuda")[:copies] if apart else torch.arange(copies, device="cuda") + 901
    x[..., top] = 9.5
    x = x.to(TYPES[name])
    order = torch.rand(64, beams, v, generator=r, device="cuda")  # a beam's own order of the other tokens, so its own roundings
    rest = torch.ones(v, dtype=torch.bool, device="cuda")
    rest[top] = False
    both = x.expand(64, beams, v).clone()
    both[..., rest] = both[..., rest].gather(2, order[..., rest].argsort(-1))
    s = torch.full((64, beams), -(2.0 ** -6), device="cuda")
    s += torch.arange(beams, device="cuda") * 2.0 ** -26 * torch.where(torch.rand(64, 1, generator=r, device="cuda") < 0.5, -1.0, 1.0)
    assert all(bool((s[:, i] != s[:, i + 1]).all()) for i in range(beams - 1))
    check(qb, both, s, k)


@pytest.mark.parametrize("name", TYPES)
@pytest.mark.parametrize("share", [0.5, 0.999, 1.0])
@pytest.mark.parametrize("k", [1, 20, 64])
def test_forbidden_tokens(qb, name, share, k):
    """Logits of -inf, until fewer than k are left, or none in a beam, or none at all: the rest in order of places."""
    x, s = make(3, 4, 9000, name, seed=3)
    x.masked_fill_(torch.rand(x.shape, generator=torch.Generator(device="cuda").manual_seed(9), device="cuda") < share, -INF)
    x[1, 2] = -INF
    check(qb, x, s, k)


@pytest.mark.parametrize("name", TYPES)
def test_lowest_numbers_of_the_type(qb, name):
    """A mask of the type's lowest value: ordinary, very small logits."""
    x, s = make(2, 3, 4000, name, seed=4)
    x[:, :, 10:3990] = torch.finfo(TYPES[name]).min
    check(qb, x, s, 30)
    x[:] = torch.finfo(TYPES[name]).min
    check(qb, x, s, 30)
    x[:] = torch.finfo(TYPES[name]).max
    check(qb, x, s, 30)


@pytest.mark.parametrize("name", TYPES)
@pytest.mark.parametrize("bad", [math.nan, INF])
def test_rows_that_are_no_numbers(qb, name, bad):
    x, s = make(2, 3, 5000, name, seed=5)
    x[0, 1, 4321] = bad
    check(qb, x, s, 12)
    x[0, :, 17] = bad
    check(qb, x, s, 12)


@pytest.mark.parametrize("bad", [math.nan, INF, -INF])
def test_beams_without_a_score(qb, bad):
    """A search's first step: one beam has a score."""
    x, s = make(2, 4, 3000, "f32", seed=6)
    s[:, 1:] = bad
    check(qb, x, s, 8)
    s[1] = bad
    check(qb, x, s, 8)


@pytest.mark.parametrize("name", TYPES)
@pytest.mark.parametrize("kind", [torch.bool, torch.uint8])
def test_ended_beams(qb, name, kind):
    x, s = make(4, 3, 2500, name, seed=7)
    s[0, 1] = 0.5  # an ended beam that is better than all else
    ended = torch.zeros(4, 3, dtype=kind, device="cuda")
    ended[0, 1] = ended[1] = ended[2, 0] = ended[2, 2] = 1
    for end_id in (0, 2, 2499):
        check(qb, x, s, 6, ended, end_id)
    x[1] = math.nan  # not looked at
    s[1, 2] = -INF
    check(qb, x, s, 64, ended, 5)


def test_rows_past_32_bits(qb):
    """Row offsets beyond 2^32 bytes and 2^31 elements."""
    v, far = 3000, (1 << 27) + 24
    buf = torch.empty(17 * far + v, device="cuda", dtype=torch.float16)
    x = buf.as_strided((6, 3, v), (3 * far, far, 1))
    x.copy_(torch.randn(6, 3, v, generator=torch.Generator(device="cuda").manual_seed(8), device="cuda"))
    check(qb, x, torch.zeros(6, 3, device="cuda"), 7)


def test_streams_graphs_and_one_object_for_many_sizes(qb):
    sel = qb.BeamSelector(8)
    side = torch.cuda.Stream()
    for g, b, v in ((2, 4, 40000), (64, 4, 30000), (1, 2, 100), (200, 1, 9000)):
        x, s = make(g, b, v, "bf16", seed=g)
        check(qb, x, s, 8, select=sel)
        want = sel(x, s)
        torch.cuda.synchronize()
        for stream in (side, side.cuda_stream, 0):
            got = sel(x, s, stream=stream)
            torch.cuda.synchronize()
            assert all(torch.equal(a, w) for a, w in zip(got, want))
    x, s = make(3, 4, 20000, "f32", seed=50)
    xs, ss = x.clone(), s.clone()
    with torch.cuda.stream(side):
        sel(xs, ss)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        out = sel(xs, ss)
    big, bs = make(200, 8, 60000, "bf16", seed=51)
    with torch.cuda.stream(side):  # a larger workspace on the same stream leaves the graph's alone
        sel(big, bs)
    for seed in (52, 53):
        x2, s2 = make(3, 4, 20000, "f32", seed=seed)
        torch.cuda.synchronize()
        xs.copy_(x2)
        ss.copy_(s2)
        graph.replay()
        torch.cuda.synchronize()
        want = expected(x2, s2, 8)
        assert torch.equal(out[1], want[1]) and torch.equal(out[2], want[2])


def test_results_do_not_depend_on_timing(qb):
    x, s = make(16, 8, 50257, "bf16", seed=60)
    sel = qb.BeamSelector(16)
    first = [t.clone() for t in sel(x, s)]
    for _ in range(50):
        assert all(torch.equal(a, b) for a, b in zip(sel(x, s), first))


def test_what_is_refused(qb):
    x, s = make(2, 3, 100, "f32")
    sel = qb.BeamSelector(4)
    e = torch.zeros(2, 3, dtype=torch.bool, device="cuda")
    for a in ((x.double(), s), (x.cpu(), s), (x[0], s), (x.transpose(1, 2), s), (x, s.half()), (x, s[:1]), (x, s.cpu()), (x, s.t()),
              (x, s, e.int()), (x, s, e[:1]), (x, s, e.cpu()), (torch.zeros(4, 3, 100, device="cuda")[::2], s)):
        with pytest.raises(TypeError):
            sel(*a)
    with pytest.raises(qb.QntError, match="end_id"):
        sel(x, s, e)
    with pytest.raises(qb.QntError, match="fewer than k"):
        qb.BeamSelector(64)(x[:, :1, :60], s[:, :1].contiguous())
    with pytest.raises(qb.QntError, match="at most 64"):
        qb.BeamSelector(65)(x, s)
    out = sel(x[:0], s[:0])
    assert all(t.shape == (0, 4) for t in out)


@pytest.mark.parametrize("k, end_id, word", [(2 ** 32 + 4, -1, "at most 64"), (-(2 ** 32) + 4, -1, "positive"), (4, 2 ** 32 + 5, "end_id"),
                                             (4, -(2 ** 32) + 5, "end_id")])
def test_numbers_past_32_bits_are_refused(qb, k, end_id, word):
    """Not taken for what their lower half says."""
    x, s = make(2, 3, 100, "f32")
    with pytest.raises(qb.QntError, match=word):
        qb.BeamSelector(k, end_id=end_id)(x, s, torch.zeros(2, 3, dtype=torch.bool, device="cuda"))


def test_two_streams_at_once(qb):
    """One object on two streams, with sizes that make both calls overlap."""
    sel, streams = qb.BeamSelector(8), [torch.cuda.Stream() for _ in range(2)]
    sets = [make(64, 4, 50000, "bf16", seed=70 + i) for i in range(2)]
    want = [sel(*a) for a in sets]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(10):
        for i in range(2):
            got[i].append(sel(*sets[i], stream=streams[i]))
    torch.cuda.synchronize()
    for i in range(2):
        for out in got[i]:
            assert all(torch.equal(a, b) for a, b in zip(out, want[i]))
