"""CPU checks of the calls on the paged KV cache: addresses that a kernel could not read are refused before any device work."""
import ctypes as C

import pytest

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
