"""CPU checks of the calls on the paged KV cache: addresses that a kernel could not read are refused before any device work, and
the workspace that a call is told to bring is the one it takes."""
import contextlib
import ctypes as C
import os
import subprocess
import sys
import types

import pytest

from conftest import ROOT
from test_kv_cache_abi import AT, INVALID, cache, refused


@pytest.mark.parametrize("array", ["scales", "refs", "table", "lens", "status"])
def test_arrays_are_aligned_to_their_elements(qb, array):
    c = cache(qb, **{array: AT + 2})
    refused(qb, qb.lib().qnt_kv_free(C.byref(c), AT, 1, None), INVALID, "aligned")
    refused(qb, qb.lib().qnt_kv_check(C.byref(c), None), INVALID, "aligned")


@pytest.mark.parametrize("dtype, off", [(0, 1), (0, 2), (1, 1), (4, 1)])
def test_rows_are_aligned_to_their_elements(qb, dtype, off):
    L, c = qb.lib(), cache(qb)
    p = C.byref(c)
    refused(qb, L.qnt_kv_append(p, 0, AT + off, AT, dtype, 128, 128, AT, AT, 1, 1, 1, None), INVALID, "aligned")
    refused(qb, L.qnt_kv_append(p, 0, AT, AT + off, dtype, 128, 128, AT, AT, 1, 1, 1, None), INVALID, "aligned")
    refused(qb, L.qnt_kv_attention(p, 0, AT + off, dtype, 128, 2, AT, AT, 1, 1, 1, 1, 1.0, 0, AT, None, AT, 1 << 30, None), INVALID,
            "aligned")
    refused(qb, L.qnt_kv_attention(p, 0, AT, dtype, 128, 2, AT, AT, 1, 1, 1, 1, 1.0, 0, AT, AT + 2, AT, 1 << 30, None), INVALID,
            "aligned")


def test_lists_are_aligned_to_their_elements(qb):
    L, c = qb.lib(), cache(qb)
    p, odd = C.byref(c), AT + 2
    for seqs, starts in ((odd, AT), (AT, odd)):
        refused(qb, L.qnt_kv_append(p, 0, AT, AT, 0, 128, 128, seqs, starts, 1, 1, 1, None), INVALID, "aligned")
        refused(qb, L.qnt_kv_attention(p, 0, AT, 0, 128, 2, seqs, starts, 1, 1, 1, 1, 1.0, 0, AT, None, AT, 1 << 30, None), INVALID, "aligned")
        refused(qb, L.qnt_kv_read(p, 0, seqs, AT, starts, 1, 1, AT, AT, 0, None), INVALID, "aligned")
        refused(qb, L.qnt_kv_reserve(p, seqs, starts, 1, AT, 1 << 30, None), INVALID, "aligned")
        refused(qb, L.qnt_kv_fork(p, seqs, starts, 1, AT, 1 << 30, None), INVALID, "aligned")
        refused(qb, L.qnt_kv_copy(p, seqs, starts, 1, None), INVALID, "page list")
    refused(qb, L.qnt_kv_read(p, 0, AT, odd, AT, 1, 1, AT, AT, 0, None), INVALID, "aligned")
    refused(qb, L.qnt_kv_free(p, odd, 1, None), INVALID, "aligned")


# In a process that sees no GPU, whatever the machine: a call that is not refused for its workspace ends with CUDA's own error.
DEMANDS = """
import ctypes as C, itertools, sys
sys.path[:0] = {paths!r}
import quanta_b200 as qb
from test_kv_cache_abi import AT, cache
L, short, calls = qb.lib(), [], 0
for (kv, group, hd), (n, m), page in itertools.product([(8, 4, 128), (2, 7, 64), (1, 1, 64), (1, 40, 128), (2, 2, 64)],
                                                       [(1, 1), (1, 4), (8, 1), (64, 1), (256, 1), (5, 2), (3, 60), (40, 300)], [16, 64]):
    for max_len in [1, 100, 128, 896, 897, 1000, 1023, 1024, 1025, 1152, 1153, 4096, 4200, 8000, 70000]:
        c = cache(qb, n_kv_heads=kv, head_dim=hd, page_tokens=page, max_seqs=300, max_pages=-(-max_len // page) + 5)
        p = C.byref(c)
        have = L.qnt_kv_attention_workspace(p, kv * group, n, n * m, m, max_len)
        for window in sorted({{0, 1, 100, 128, 900, 1000, 1023, 4096, 8192, max_len - 1, max_len, max_len + 1, max_len - m, max_len + 79,
                              max_len + 200, 2 ** 31 - 1}} - {{-1}} - set(range(-400, 0))):
            for dtype in (0, 1, 4):
                rc = L.qnt_kv_attention(p, 0, AT, dtype, kv * group * hd, kv * group, AT, AT, n, n * m, m, max_len, 1.0, window, AT, None,
                                        AT, have, None)
                calls += 1
                why = L.qnt_last_error().decode()
                assert rc != 0, "a GPU was seen"
                if "workspace" in why:
                    short.append((kv, group, hd, n, m, max_len, window, dtype, have, why))
print(calls, len(short), short[:5])
sys.exit(1 if short else 0)
"""


def test_the_workspace_that_is_asked_for_is_enough_with_any_window(qb):
    paths = [str(ROOT / "quanta.cpp_b200"), str(ROOT / "tests")]
    r = subprocess.run([sys.executable, "-c", DEMANDS.format(paths=paths)], env=dict(os.environ, CUDA_VISIBLE_DEVICES=""), capture_output=True,
                       text=True, timeout=600)
    assert r.returncode == 0, r.stdout[-2000:] + r.stderr[-2000:]


class FakeCuda:
    def __init__(self):
        self.now = 0

    def current_device(self):
        return self.now

    @contextlib.contextmanager
    def device(self, index):
        was, self.now = self.now, index
        yield
        self.now = was


def on(index, dtype, shape=(4,)):
    """What PagedKV looks at of a tensor on a device."""
    strides = [1] * len(shape)
    for i in range(len(shape) - 2, -1, -1):
        strides[i] = strides[i + 1] * shape[i + 1]
    return types.SimpleNamespace(dtype=dtype, shape=shape, stride=lambda: tuple(strides), is_cuda=index >= 0, get_device=lambda: index,
                                 is_contiguous=lambda: True, numel=lambda: shape[0], data_ptr=lambda: AT,
                                 device=types.SimpleNamespace(type="cuda", index=index))


def test_a_cache_on_another_device_than_the_current_one(qb):
    """Calls run on the cache's device and its stream; tensors of another device are refused.  (A second device is not needed: the
    library and torch's device are stood in for.)"""
    cuda, calls = FakeCuda(), []

    class Lib:
        def __getattr__(self, name):
            return lambda *args: calls.append((name, cuda.now, args)) or 0

    kv = qb.PagedKV.__new__(qb.PagedKV)
    kv._torch, kv._lib, kv._index, kv._raw_stream = types.SimpleNamespace(cuda=cuda), Lib(), 1, lambda i: 70 + i
    kv._current_device = cuda.current_device
    kv._i32, kv._types, kv._p, kv._page_ws = "int32", {"f16": qb.F16}, None, 64
    kv._ws, kv._kept, kv._need = {71: on(1, "uint8", (1 << 20,))}, [], {}
    kv.n_kv_heads, kv.head_dim = 2, 64
    here, there, rows = on(1, "int32"), on(0, "int32"), on(1, "f16", (3, 2, 64))
    kv.free(here)
    kv.reserve(here, here)
    kv.fork(here, here)
    kv.copy_pages(here, here)
    kv.compact()
    kv.append(0, rows, rows, on(1, "int32", (3,)), here)
    kv.check()
    assert [c[0] for c in calls] == ["qnt_kv_" + n for n in "free reserve fork copy compact append check".split()]
    assert all(now == 1 and args[-1] == 71 for _, now, args in calls) and cuda.now == 0
    n = len(calls)
    for bad in (lambda: kv.free(there), lambda: kv.reserve(here, there), lambda: kv.fork(there, here), lambda: kv.free(on(-1, "int32")),
                lambda: kv.append(0, rows, on(0, "f16", (3, 2, 64)), on(1, "int32", (3,)), here),
                lambda: kv.attention(0, on(0, "f16", (3, 2, 64)), on(1, "int32", (3,)), here, 1, 9)):
        with pytest.raises(TypeError, match="device"):
            bad()
    assert len(calls) == n
