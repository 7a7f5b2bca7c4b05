"""The paged 8-bit KV cache's workspaces and outputs, with captured graphs and with work on a stream that is not the current one."""
import pytest

from test_gpu_kv_cache import ints, make, queries

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu


def test_a_graph_keeps_its_workspace(qb):
    """A captured call writes to its workspace at every replay: a larger call on the same stream leaves that memory alone."""
    c = make(qb, [5000, 4000] + [3000] * 30, 2, 64, 64, seed=50)
    side = torch.cuda.Stream()
    q, seqs, starts = queries(2, 14, 64, "f32"), ints([0, 1]), ints([0, 1, 2])
    many, all_seqs = queries(32 * 40, 14, 64, "f32"), ints(range(32))
    all_starts = ints(range(0, 32 * 40 + 1, 40))
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        want = c.attention(0, q, seqs, starts, 1, 5000)
    torch.cuda.synchronize()
    old = c._ws[side.cuda_stream]
    at, size = old.data_ptr(), old.numel()
    del old
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=side):
        out = c.attention(0, q, seqs, starts, 1, 5000)
    with torch.cuda.stream(side):
        c.attention(0, many, all_seqs, all_starts, 40, 5000)
    torch.cuda.synchronize()
    assert c._ws[side.cuda_stream].numel() > size
    with torch.cuda.stream(side):  # what the allocator would give away, it gives here
        taken = [torch.full((size,), 7, dtype=torch.uint8, device="cuda") for _ in range(8)]
    torch.cuda.synchronize()
    assert all(t.data_ptr() + size <= at or t.data_ptr() >= at + size for t in taken)
    for _ in range(2):
        out.zero_()
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want)
    assert all(bool((t == 7).all()) for t in taken)
    c.check()


@pytest.mark.parametrize("call", ["attention", "read"])
def test_outputs_on_a_stream_of_their_own(qb, call):
    """With stream=, nothing that the current stream still has queued reaches the outputs."""
    c = make(qb, [2000] * 8, 2, 64, 64, seed=51)
    side = torch.cuda.Stream()
    q, seqs, starts = queries(8, 14, 64, "f32"), ints(range(8)), ints(range(9))
    rows, first = ints(range(0, 801, 100)), ints([0] * 8)
    run = {"attention": lambda s: c.attention(0, q, seqs, starts, 1, 2000, lse=True, stream=s),
           "read": lambda s: c.read(0, seqs, first, rows, 800, stream=s)}[call]
    want = [x.clone() for x in run(None)]
    run(side)  # (the side stream's workspace)
    torch.cuda.synchronize()
    shapes = [x.shape for x in want]
    for _ in range(3):
        blocks = [torch.empty(s, device="cuda") for s in shapes for _ in range(4)]
        torch.cuda._sleep(20_000_000)  # about 10 ms: the fills below are still queued when the call runs
        for b in blocks:
            b.fill_(7.0)
        del b, blocks
        got = run(side)
        torch.cuda.synchronize()
        for a, w in zip(got, want):
            assert torch.equal(a, w)
    by_number = run(side.cuda_stream)
    torch.cuda.synchronize()
    assert all(torch.equal(a, w) for a, w in zip(by_number, want))
    torch.cuda.synchronize()
    on_default = run(0)  # the legacy default stream
    torch.cuda.synchronize()
    assert all(torch.equal(a, w) for a, w in zip(on_default, want))
