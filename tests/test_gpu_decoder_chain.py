"""The operators around a decoder layer and a beam search right behind each other on one stream, each reading in its first instructions
what the one before wrote last, buffers reused: every call starts only where its inputs are complete."""
import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("captured", [False, True])
@pytest.mark.parametrize("m", [1, 70, 6000])
def test_norm_values_and_rotations_in_a_row(qb, m, captured):
    g = torch.Generator(device="cuda").manual_seed(m)
    x, w = torch.randn(m, 1024, generator=g, device="cuda").half(), torch.rand(1024, generator=g, device="cuda") + 0.5
    rope, pos = qb.Rope(64), torch.randint(0, 5000, (m,), generator=g, device="cuda", dtype=torch.int32)

    def layer(v, res, sync):
        for _ in range(6):
            q8, d = qb.rms_norm_q8(v, w, residual=res)
            sync()
            v = qb.dequantize_q8(q8, d, torch.float16)
            sync()
            q, k = rope(v[:, :768].unflatten(1, (12, 64)), v[:, 768:].unflatten(1, (4, 64)), pos)
            sync()
            rope(q, k, pos, inplace=True)
            sync()
            v = torch.cat([q.flatten(1), k.flatten(1)], 1)
        return v

    res = torch.zeros(m, 1024, device="cuda")
    want = layer(x, res, torch.cuda.synchronize)
    kept = res.clone()
    if captured:
        r2, graph = torch.zeros_like(res), torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = layer(x, r2, lambda: None)
        for _ in range(5):
            r2.zero_()
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(out, want) and torch.equal(r2, kept)
    else:
        for _ in range(5):
            r2 = torch.zeros_like(res)
            out = layer(x, r2, lambda: None)
            torch.cuda.synchronize()
            assert torch.equal(out, want) and torch.equal(r2, kept)


@pytest.mark.parametrize("captured", [False, True])
@pytest.mark.parametrize("g, b, v", [(1, 4, 900), (40, 8, 20000)])
def test_selections_in_a_row(qb, g, b, v, captured):
    """Each selection's scores and ended beams are the last one's results, copied into the same buffers."""
    r = torch.Generator(device="cuda").manual_seed(v)
    x = [torch.randn(g, b, v, generator=r, device="cuda").bfloat16() for _ in range(3)]
    sel = qb.BeamSelector(b, end_id=0)
    s, e = torch.zeros(g, b, device="cuda"), torch.zeros(g, b, dtype=torch.bool, device="cuda")

    def steps(sync):
        s.copy_(-torch.arange(b, device="cuda").float().expand(g, b))
        e.zero_()
        got = []
        for i in range(12):
            scores, tokens, parents = sel(x[i % 3], s, e)
            sync()
            s.copy_(scores)
            e.copy_((tokens % 7 == 0) & (i < 8))
            sync()
            got += [scores, tokens, parents]
        return got

    want = [t.clone() for t in steps(torch.cuda.synchronize)]
    if captured:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = steps(lambda: None)
        for _ in range(5):
            graph.replay()
            torch.cuda.synchronize()
            assert all(torch.equal(a, w) for a, w in zip(out, want))
    else:
        for _ in range(5):
            out = steps(lambda: None)
            torch.cuda.synchronize()
            assert all(torch.equal(a, w) for a, w in zip(out, want))
