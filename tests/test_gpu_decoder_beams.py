"""A beam search over a decoder made of the public operators: norm, quantized products, rotary positions, the paged cache's append
and attention, the selection, the reordering.

What is checked at the end of every step: each sequence's first layer's keys are those of the tokens that its beam has taken, traced
through the parents on the host.  A key is rope(W norm(embedding)): the norm's rounding moves a code by at most one of 127 (0.5 for
the rounding itself, which the definition has too), the product adds cols / 32 = 8 f32 roundings a block, the rotation 1.2e-6, the
cache half a code of its block.  So |key - exact| <= sum_i |w_i| d_i 1.001 (every code one off) is far too wide; the definition is
therefore taken from the codes that the norm gave, which test_gpu_decoder_rows.py checks.  An append that brings a larger value
than its block holds rounds the block's earlier codes again, by at most half of the new scale, and no scale is above the last one, d:
with r later appends of that kind |key - definition| <= (0.5 (1 + r) + 0.01) d + 2^-18 sum_i |w_i q_i| d_i (the 0.01: f32 roundings of
codes up to 127)."""
import ctypes as C
import math

import numpy as np
import pytest

from test_gpu_kv_cache import ints, values

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

DIM, HEADS, KV, HD, FFN, VOCAB, LAYERS = 256, 4, 2, 64, 512, 777, 2


class Weight:
    """A Q8_0 matrix on the device and its values."""

    def __init__(self, qb, rows, cols, rng):
        q = rng.integers(-127, 128, (rows, cols)).astype(np.int8)
        d = (rng.random((rows, cols // 32)) * 0.8 + 0.2).astype(np.float16) * np.float16(0.02 / 64)
        self.t = qb.DeviceTensor(qb.Q8_0, rows, cols, q.tobytes() + d.tobytes())
        self.rows, self.lib = rows, qb.lib()
        self.values = torch.from_numpy(q.astype(np.float64) * np.repeat(d.astype(np.float64), 32, 1)).cuda()

    def __call__(self, q, d):
        out = torch.empty(q.shape[0], self.rows, device="cuda")
        st = torch.cuda.current_stream().cuda_stream
        rc = self.lib.qnt_matmul(self.t.h, q.data_ptr(), d.data_ptr(), q.shape[0], 0, self.rows, out.data_ptr(), self.rows, 1, st)
        assert rc == 0, self.lib.qnt_last_error()
        return out


def quantized(qb, x):
    q = torch.empty(x.shape, dtype=torch.int8, device="cuda")
    d = torch.empty(x.shape[0], x.shape[1] // 32, device="cuda")
    assert qb.lib().qnt_quantize_q8(x.data_ptr(), x.shape[0], x.shape[1], q.data_ptr(), d.data_ptr(),
                                    torch.cuda.current_stream().cuda_stream) == 0
    return q, d


class Decoder:
    def __init__(self, qb, seed):
        rng = np.random.default_rng(seed)
        g = torch.Generator(device="cuda").manual_seed(seed)
        self.qb, self.rope = qb, qb.Rope(HD, base=1e4, scaling=dict(kind="linear", factor=2.0))
        self.embed = torch.randn(VOCAB, DIM, generator=g, device="cuda")
        self.norms = 1 + 0.2 * torch.randn(2 * LAYERS + 1, DIM, generator=g, device="cuda")
        self.qkv = [Weight(qb, (HEADS + 2 * KV) * HD, DIM, rng) for _ in range(LAYERS)]
        self.o = [Weight(qb, DIM, HEADS * HD, rng) for _ in range(LAYERS)]
        self.up = [Weight(qb, FFN, DIM, rng) for _ in range(LAYERS)]
        self.down = [Weight(qb, DIM, FFN, rng) for _ in range(LAYERS)]
        self.head = Weight(qb, VOCAB, DIM, rng)

    def keys(self, tokens, positions):
        """Layer 0's keys of tokens at positions: the definition in 64 bits from the norm's codes, and sum |w q| d."""
        q, d = self.qb.rms_norm_q8(self.embed[tokens], self.norms[0], 1e-6)
        x = self.qb.dequantize_q8(q, d, torch.float32).double()
        w = self.qkv[0].values[HEADS * HD: (HEADS + KV) * HD]
        k, mag = (x @ w.T).view(-1, KV, HD), (x.abs() @ w.abs().T).view(-1, KV, HD)
        f = torch.tensor(self.qb.Rope.frequencies(HD, 1e4, dict(kind="linear", factor=2.0))[0], dtype=torch.float64, device="cuda")
        a = positions.double()[:, None, None] * f
        lo, hi = k[..., : HD // 2], k[..., HD // 2:]
        m = mag[..., : HD // 2] + mag[..., HD // 2:]
        return torch.cat([lo * a.cos() - hi * a.sin(), lo * a.sin() + hi * a.cos()], -1), torch.cat([m, m], -1)

    def logits(self, kv, tokens, positions, seqs, starts, max_q, max_len):
        r = torch.zeros(tokens.numel(), DIM, device="cuda")
        x = self.embed[tokens.long()]
        for l in range(LAYERS):
            rows = self.qkv[l](*self.qb.rms_norm_q8(x, self.norms[2 * l], 1e-6, residual=r)).view(-1, HEADS + 2 * KV, HD)
            q, k = self.rope(rows[:, :HEADS], rows[:, HEADS: HEADS + KV], positions)
            kv.append(l, k, rows[:, HEADS + KV:], seqs, starts, max_q)
            a = kv.attention(l, q, seqs, starts, max_q, max_len)
            x = self.o[l](*quantized(self.qb, a.view(-1, HEADS * HD)))
            u = self.up[l](*self.qb.rms_norm_q8(x, self.norms[2 * l + 1], 1e-6, residual=r))
            x = self.down[l](*quantized(self.qb, torch.nn.functional.silu(u)))
        last = starts[1:].long() - 1
        r, x = r[last], x[last].contiguous()
        return self.head(*self.qb.rms_norm_q8(x, self.norms[-1], 1e-6, residual=r))


def roundings(keys, first):
    """For each position and head: 1 + the later appends that bring a larger value into its block (16 positions).  The first `first`
    positions came in one append, the others in one each; a value within a thousandth of the largest counts as larger."""
    top = keys.abs().amax(-1).cpu().numpy()  # [len][heads]
    out = np.ones_like(top)
    for b in range(0, len(top), 16):
        end = min(b + 16, len(top))
        calls = [range(b, min(first, end))] if b < first else []
        calls += [range(p, p + 1) for p in range(max(first, b), end)]
        most = np.zeros(top.shape[1])
        for k, c in enumerate(calls):
            new = top[c].max(0)
            if k:
                out[b: c[0]] += new > most * 0.999
            most = np.maximum(most, new)
    return torch.from_numpy(out).cuda()[..., None]


@pytest.mark.parametrize("lens, beams, steps", [([7, 40, 33], 4, 12), ([90], 7, 20)])
def test_beam_search_over_a_decoder_of_operators(qb, lens, beams, steps):
    m, groups = Decoder(qb, 3), len(lens)
    n = groups * beams
    rng = np.random.default_rng(5)
    kv = qb.PagedKV.empty(LAYERS, KV, HD, n * 8 + 20, n, 8, 16)
    prompts = [rng.integers(0, VOCAB, k).tolist() for k in lens]
    first = ints(range(0, n, beams))
    starts = ints([0] + list(np.cumsum(lens)))
    kv.reserve(first, ints(lens))
    flat = ints(sum(prompts, []))
    pos = ints(sum((list(range(k)) for k in lens), []))
    logits = m.logits(kv, flat, pos, first, starts, max(lens), max(lens))
    select_first, select = qb.BeamSelector(beams), qb.BeamSelector(beams)
    scores, tokens, parents = select_first(logits.view(groups, 1, VOCAB), torch.zeros(groups, 1, device="cuda"))
    others = [s for s in range(n) if s % beams]
    kv.fork(ints([s - s % beams for s in others]), ints(others))
    seqs, ones, every = ints(range(n)), ints([1] * n), ints(range(n + 1))
    told = [[p + [int(tokens[g, b])] for b in range(beams)] for g, p in enumerate(prompts)]  # the last one is not in the cache yet
    total = scores.double().cpu().numpy()
    for step in range(steps):
        kv.reserve(seqs, ones)
        positions = kv.lens[:n] - 1
        logits = m.logits(kv, tokens.view(-1), positions, seqs, every, 1, max(lens) + steps)
        before = scores
        scores, tokens, parents = select(logits.view(groups, beams, VOCAB), scores)
        kv.reorder(seqs, parents, beams)
        lp = torch.log_softmax(logits.double(), -1).view(groups, beams, VOCAB)
        for g in range(groups):
            told[g] = [told[g][int(parents[g, b])] + [int(tokens[g, b])] for b in range(beams)]
            total[g] = [total[g][int(parents[g, b])] + float(lp[g, parents[g, b], tokens[g, b]]) for b in range(beams)]
        best = (before.double()[..., None] + lp).flatten(1).topk(beams).values
        assert bool(((scores.double() - best).abs() <= 3e-6 + 2.0 ** -24 * best.abs()).all())
        for s in range(n):
            mine = told[s // beams][s % beams][:-1]
            t = torch.tensor(mine, device="cuda")
            want, mag = m.keys(t, torch.arange(len(mine), device="cuda"))
            got = values(kv, 0, s)[0]
            assert got.shape[0] == len(mine) == int(kv.lens[s])
            pages = kv.table[s, : -(-len(mine) // 16)].long()
            d = kv.scales[pages, 0, 0].double()[..., 0].repeat_interleave(16, 0)[: len(mine), :, None]  # a page is a block here
            again = roundings(want, lens[s // beams])
            assert bool(((got - want).abs() <= (0.5 * again + 0.01) * d + 2.0 ** -18 * mag).all()), (step, s)
    kv.check()
    for g in range(groups):
        assert len({tuple(x) for x in told[g]}) == beams
        assert np.all(np.abs(scores[g].cpu().numpy() - total[g]) <= (steps + 1) * (3e-6 + 2.0 ** -23 * np.abs(total[g])))
    kv.free(seqs)
    kv.check()
    assert not kv.refs.any()


def test_a_step_in_a_graph(qb):
    """Reserve, decode, select and reorder captured once and replayed: the same as queued one by one."""
    m, beams = Decoder(qb, 4), 4
    prompt = np.random.default_rng(6).integers(0, VOCAB, 50).tolist()

    def fresh():
        kv = qb.PagedKV.empty(LAYERS, KV, HD, 60, beams, 8, 16)
        kv.reserve(ints([0]), ints([50]))
        logits = m.logits(kv, ints(prompt), ints(range(50)), ints([0]), ints([0, 50]), 50, 50)
        s, t, _ = qb.BeamSelector(beams)(logits.view(1, 1, VOCAB), torch.zeros(1, 1, device="cuda"))
        kv.fork(ints([0] * 3), ints([1, 2, 3]))
        return kv, s.clone(), t.clone()

    def step(kv, sel, scores, tokens):
        kv.reserve(seqs, ones)
        logits = m.logits(kv, tokens.view(-1), kv.lens - 1, seqs, every, 1, 128)
        s, t, p = sel(logits.view(1, beams, VOCAB), scores)
        kv.reorder(seqs, p)
        scores.copy_(s)
        tokens.copy_(t)

    seqs, ones, every = ints(range(4)), ints([1] * 4), ints(range(5))
    kv, scores, tokens = fresh()
    sel = qb.BeamSelector(beams)
    for _ in range(8):
        step(kv, sel, scores, tokens)
    kv.check()
    kv2, scores2, tokens2 = fresh()
    sel2 = qb.BeamSelector(beams)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(kv2, sel2, scores2, tokens2)  # (makes the workspaces)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=side):
        step(kv2, sel2, scores2, tokens2)
    for _ in range(7):
        g.replay()
    torch.cuda.synchronize()
    kv2.check()
    assert torch.equal(tokens, tokens2) and torch.equal(scores, scores2) and torch.equal(kv.table, kv2.table)
    assert math.isfinite(float(scores.sum()))
