"""Calls of the operators on torch tensors that are refused, or that others have to notice: counts past 32 bits, tensors
that the call writes in place, calls from several threads."""
import threading
import time

import pytest

from test_gpu_kv_cache import ints

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

MANY = 1 << 31


def test_more_tokens_than_a_call_takes(qb):
    """2^31 tokens are not 2^31 - 1: refused, nothing is written."""
    x, pos = torch.ones(MANY, 1, 2, dtype=torch.float16, device="cuda"), torch.ones(MANY, dtype=torch.int32, device="cuda")
    with pytest.raises(ValueError, match="2147483647"):
        qb.Rope(2)(x, None, pos, inplace=True)
    assert bool((x[:3] == 1).all()) and bool((x[-3:] == 1).all())
    del x
    one = torch.ones(1, 2, dtype=torch.float16, device="cuda").expand(MANY, 1, 2)
    with pytest.raises(ValueError, match="2147483647"):
        qb.Rope(2)(one, None, pos)
    del pos
    with pytest.raises(ValueError, match="2147483647"):
        qb.rms_norm_q8(torch.ones(32, device="cuda").expand(MANY, 32), torch.ones(32, device="cuda"))


class InPlace:
    """The calls that write one of their arguments: (call, tensors that it writes)."""

    def __init__(self, qb):
        self.x, self.w = torch.randn(4, 64, device="cuda"), torch.ones(64, device="cuda")
        self.pos, rope = torch.arange(4, device="cuda", dtype=torch.int32), qb.Rope(16)
        self.calls = {"residual": lambda t: qb.rms_norm_q8(self.x, self.w, residual=t),
                      "q": lambda t: rope(t.view(4, 4, 16), None, self.pos, inplace=True),
                      "k": lambda t: rope(self.x.view(4, 4, 16).clone(), t.view(4, 4, 16), self.pos, inplace=True)}


@pytest.mark.parametrize("which", ["residual", "q", "k"])
def test_writes_in_place_are_seen_by_autograd(qb, which):
    call = InPlace(qb).calls[which]
    leaf = torch.randn(4, 64, device="cuda", requires_grad=True)
    kept = leaf.detach().clone()
    with pytest.raises(RuntimeError, match="gradient"):
        call(leaf)
    with pytest.raises(RuntimeError, match="gradient"):
        call(leaf * 1.0)
    assert torch.equal(leaf, kept)
    # where no gradients are recorded the call goes through, and what was saved before it is known to be stale
    y = (leaf * 1.0).exp()
    before = y._version
    with torch.no_grad():
        call(y)
    assert y._version > before
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.sum().backward()
    plain = torch.randn(4, 64, device="cuda")
    before = plain._version
    call(plain)
    assert plain._version > before
    with torch.inference_mode():
        call(torch.randn(4, 64, device="cuda"))


def test_tangents_of_what_is_written_are_not_lost(qb):
    calls, fw = InPlace(qb).calls, torch.autograd.forward_ad
    with fw.dual_level():
        t = fw.make_dual(torch.randn(4, 64, device="cuda"), torch.ones(4, 64, device="cuda"))
        for call in calls.values():
            with pytest.raises(RuntimeError, match="gradient"):
                call(t)


@pytest.mark.parametrize("side", [0, 64])
def test_operands_side_by_side_in_one_buffer(qb, side):
    """Rows of x beside those of the residual, heads rotated in place beside each other: not the overlap that is refused."""
    buf = torch.randn(50, 128, device="cuda")
    x, r = buf[:, side: side + 64], buf[:, 64 - side: 128 - side]
    want = x + r
    qb.rms_norm_q8(x, torch.ones(64, device="cuda"), residual=r)
    assert torch.equal(r, want)
    rope, pos = qb.Rope(16), torch.arange(50, device="cuda", dtype=torch.int32)
    q, k = x.unflatten(1, (4, 16)), r.unflatten(1, (4, 16))
    want = rope(q, k, pos)
    got = rope(q, k, pos, inplace=True)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1]) and got[0].data_ptr() == x.data_ptr()
    with pytest.raises(qb.QntError, match="overlap"):
        rope(q, q, pos, inplace=True)
    with pytest.raises(qb.QntError, match="overlap"):
        rope(q[:49], q[1:], pos[:49], inplace=True)
    with pytest.raises(qb.QntError, match="overlap"):
        qb.rms_norm_q8(buf[:-1, :64], torch.ones(64, device="cuda"), residual=buf[1:, :64])


def test_a_table_that_is_not_the_rotations(qb):
    """A Rope whose table or size a caller has replaced: refused, nothing is read past its end."""
    x, pos = torch.randn(3, 2, 128, device="cuda"), torch.arange(3, device="cuda", dtype=torch.int32)
    for change in (dict(rotary_dim=128), dict(rotary_dim=66), dict(rotary_dim=32), dict(rotary_dim=-64), dict(turns=qb.Rope(64).turns.float()),
                   dict(turns=qb.Rope(64).turns.cpu()), dict(turns=qb.Rope(128).turns[::2]), dict(turns=None)):
        rope = qb.Rope(64)
        for name, value in change.items():
            setattr(rope, name, value)
        with pytest.raises(TypeError, match="turns"):
            rope(x, None, pos)


def test_reordering_and_reserving_from_threads(qb):
    """Caches whose plans need different amounts of shared memory, each on a thread of its own (the C calls leave Python's lock)."""
    wrong = []

    def work(pages, calls):
        try:
            torch.cuda.set_device(0)
            stream = torch.cuda.Stream()
            with torch.cuda.stream(stream):
                c = qb.PagedKV.empty(1, 1, 64, pages, 4, 4, 16)
                seqs, parents, none = ints([0, 1]), ints([0, 1]), ints([0, 0])
                ws = torch.empty(qb.lib().qnt_kv_reorder_workspace(c._p) + c._page_ws, dtype=torch.uint8, device="cuda")
                for _ in range(calls):
                    for rc in (qb.lib().qnt_kv_reorder(c._p, seqs.data_ptr(), parents.data_ptr(), 2, 2, ws.data_ptr(), ws.numel(),
                                                       stream.cuda_stream),
                               qb.lib().qnt_kv_reserve(c._p, seqs.data_ptr(), none.data_ptr(), 2, ws.data_ptr(), ws.numel(),
                                                       stream.cuda_stream)):
                        if rc:
                            wrong.append((pages, rc, qb.lib().qnt_last_error()))
                            return
                c.check()
        except Exception as e:
            wrong.append(repr(e))

    threads = [threading.Thread(target=work, args=(p, 6000)) for p in (280_000, 1_000_000, 400_000)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not wrong, wrong


@pytest.mark.parametrize("which", ["norm", "values", "rope", "beams", "reorder"])
def test_a_full_queue_does_not_stop_other_threads(qb, which):
    """A call that waits for room in the GPU's queue, behind half a second of other work, leaves Python's lock to others."""
    x, w, pos = torch.randn(2, 64, device="cuda"), torch.ones(64, device="cuda"), ints([0, 1])
    q8, rope, select = qb.rms_norm_q8(x, w), qb.Rope(16), qb.BeamSelector(2)
    c = qb.PagedKV.empty(1, 1, 64, 4, 2, 2, 16)
    call = {"norm": lambda: qb.rms_norm_q8(x, w), "values": lambda: qb.dequantize_q8(*q8),
            "rope": lambda: rope(x.view(2, 4, 16), None, pos), "beams": lambda: select(x.view(1, 2, 64), x[:1, :2].contiguous()),
            "reorder": lambda: c.reorder(pos, pos)}[which]
    call()
    torch.cuda.synchronize()
    stop, longest = threading.Event(), [0.0]

    def tick():
        last = time.perf_counter()
        while not stop.is_set():
            time.sleep(0.001)
            now = time.perf_counter()
            longest[0], last = max(longest[0], now - last), now

    t = threading.Thread(target=tick)
    t.start()
    began = time.perf_counter()
    torch.cuda._sleep(10 ** 9)  # (cycles)
    for _ in range(2500):
        call()
    waited = time.perf_counter() - began
    stop.set()
    t.join()
    torch.cuda.synchronize()
    assert waited > 0.3 and longest[0] < 0.5 * waited, (waited, longest)


def test_one_selector_for_two_threads_on_one_stream(qb):
    """Calls of several launches that share a workspace: those of two threads stay apart."""
    select, stream, wrong = qb.BeamSelector(4), torch.cuda.Stream(), []
    sets = [(torch.randn(8, 4, 3000, device="cuda", generator=torch.Generator(device="cuda").manual_seed(i)),
             torch.zeros(8, 4, device="cuda")) for i in range(2)]
    want = [select(*s) for s in sets]
    torch.cuda.synchronize()

    def work(i):
        try:
            with torch.cuda.stream(stream):
                got = [select(*sets[i]) for _ in range(1500)]
                stream.synchronize()
            wrong.extend(i for out in got if not all(torch.equal(a, b) for a, b in zip(out, want[i])))
        except Exception as e:
            wrong.append(repr(e))

    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not wrong, wrong[:5]
