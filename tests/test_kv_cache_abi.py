"""CPU checks of the paged KV cache's C ABI: what it refuses, with which code and message, before any device work."""
import ctypes as C

import pytest

OK, INVALID, UNSUPPORTED = 0, -1, -4
AT = 1 << 20  # a 16-byte aligned address that no call below reads


def cache(qb, **change):
    d = dict(n_layers=2, n_kv_heads=2, head_dim=64, page_tokens=64, n_pages=10, max_seqs=4, max_pages=8, codes=AT, scales=AT,
             refs=AT, table=AT, lens=AT, status=AT)
    d.update(change)
    return qb.KVCacheC(*[d[n] for n, _ in qb.KVCacheC._fields_])


def refused(qb, rc, code, word):
    assert rc == code, (rc, qb.lib().qnt_last_error())
    assert word in qb.lib().qnt_last_error().decode(), qb.lib().qnt_last_error()


@pytest.mark.parametrize("change, code, word", [
    (dict(codes=None), INVALID, "null"), (dict(status=None), INVALID, "null"), (dict(codes=AT + 8), INVALID, "aligned"),
    (dict(n_pages=0), INVALID, "positive"), (dict(max_seqs=-1), INVALID, "positive"), (dict(head_dim=96), UNSUPPORTED, "head_dim"),
    (dict(page_tokens=48), UNSUPPORTED, "page_tokens"), (dict(n_pages=(1 << 20) + 1), UNSUPPORTED, "pages"),
    (dict(max_seqs=8193), UNSUPPORTED, "sequences"), (dict(max_pages=1 << 25), UNSUPPORTED, "too long")])
def test_cache_descriptions_are_checked(qb, change, code, word):
    L, c = qb.lib(), cache(qb, **change)
    p = C.byref(c)
    refused(qb, L.qnt_kv_compact(p, AT, 1 << 30, None), code, word)
    refused(qb, L.qnt_kv_free(p, AT, 1, None), code, word)
    refused(qb, L.qnt_kv_append(p, 0, AT, AT, 0, 128, 128, AT, AT, 1, 1, 1, None), code, word)
    refused(qb, L.qnt_kv_attention(p, 0, AT, 0, 128, 2, AT, AT, 1, 1, 1, 1, 1.0, 0, AT, None, AT, 1 << 30, None), code, word)
    assert L.qnt_kv_page_workspace(p) == 0 and L.qnt_kv_attention_workspace(p, 2, 1, 1, 1, 1) == 0


def test_calls_are_checked(qb):
    L, c = qb.lib(), cache(qb)
    p = C.byref(c)

    def append(layer=0, k=AT, dtype=0, stride=128, seqs=AT, n=1, n_tok=2, max_new=2):
        return L.qnt_kv_append(p, layer, k, AT, dtype, stride, 128, seqs, AT, n, n_tok, max_new, None)

    refused(qb, append(layer=2), INVALID, "layer")
    refused(qb, append(k=None), INVALID, "null rows")
    refused(qb, append(dtype=2), UNSUPPORTED, "dtype")
    refused(qb, append(stride=127), INVALID, "stride")
    refused(qb, append(seqs=None), INVALID, "null sequence list")
    refused(qb, append(n=5), INVALID, "count")
    refused(qb, append(n_tok=-1), INVALID, "count")
    refused(qb, append(max_new=0), INVALID, "max_new")

    def attention(layer=0, q=AT, dtype=0, stride=256, heads=4, n=1, n_tok=2, max_q=2, max_len=9, window=0, out=AT, ws=AT,
                  ws_bytes=1 << 40):
        return L.qnt_kv_attention(p, layer, q, dtype, stride, heads, AT, AT, n, n_tok, max_q, max_len, 1.0, window, out, None, ws,
                                  ws_bytes, None)

    refused(qb, attention(layer=-1), INVALID, "layer")
    refused(qb, attention(q=None), INVALID, "null q")
    refused(qb, attention(out=AT + 4), INVALID, "aligned")
    refused(qb, attention(dtype=3), UNSUPPORTED, "dtype")
    refused(qb, attention(heads=5), INVALID, "n_heads")
    refused(qb, attention(heads=0), INVALID, "n_heads")
    refused(qb, attention(stride=255), INVALID, "q_stride")
    refused(qb, attention(max_q=0), INVALID, "max_q")
    refused(qb, attention(max_len=-1), INVALID, "max_len")
    refused(qb, attention(window=-1), INVALID, "window")
    refused(qb, L.qnt_kv_read(p, 0, AT, AT, AT, 1, 1, AT, AT + 8, 0, None), INVALID, "aligned")
    refused(qb, L.qnt_kv_read(p, 5, AT, AT, AT, 1, 1, AT, AT, 0, None), INVALID, "layer")
    need = L.qnt_kv_page_workspace(p)
    assert need > 0
    for f in (lambda w, b: L.qnt_kv_reserve(p, AT, AT, 1, w, b, None), lambda w, b: L.qnt_kv_fork(p, AT, AT, 1, w, b, None),
              lambda w, b: L.qnt_kv_compact(p, w, b, None)):
        refused(qb, f(AT, need - 1), INVALID, "workspace")
        refused(qb, f(None, need), INVALID, "workspace")
        refused(qb, f(AT + 8, need), INVALID, "workspace")
    refused(qb, L.qnt_kv_reserve(p, AT, None, 1, AT, need, None), INVALID, "null sequence list")
    refused(qb, L.qnt_kv_fork(p, AT, AT, 5, AT, need, None), INVALID, "count")
    refused(qb, L.qnt_kv_copy(p, AT, None, 1, None), INVALID, "page list")


def test_empty_calls_do_nothing(qb):
    L, c = qb.lib(), cache(qb)
    p = C.byref(c)
    assert L.qnt_kv_append(p, 0, None, None, 0, 0, 0, None, None, 0, 0, 0, None) == OK
    assert L.qnt_kv_read(p, 0, None, None, None, 0, 0, None, None, 0, None) == OK
    assert L.qnt_kv_attention(p, 0, None, 0, 0, 4, None, None, 0, 0, 0, 0, 1.0, 0, None, None, None, 0, None) == OK
    assert L.qnt_kv_free(p, None, 0, None) == OK and L.qnt_kv_copy(p, None, None, 0, None) == OK
    assert L.qnt_kv_attention_workspace(p, 4, 0, 0, 0, 0) == 0
