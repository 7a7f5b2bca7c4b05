"""Batched serving from the paged 8-bit KV cache (qnt_batch_init_paged / qnt_batch_fork / qnt_batch_resize).

A layer's K and V are rounded to 8 bits with a scale per 16 tokens, so the ids are not compared with the f16 caches' ones;
the last token's residual is.  The rounding's share: an element's error is uniform within half a step of amax / 127, that is
amax / 440 rms, and with amax near 4 times the rms under 1% of the values.  The residual's part that comes from the context
is at least as far from another context's as it is large, so 10% of that distance leaves a factor of ten, while one wrong
page, position or head moves the residual by about the distance itself."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu

F16, PAGED = "f16", "paged"


def residual(qb, m):
    out = np.zeros(m.hp.dim, np.float32)
    import ctypes as C
    n = qb.lib().qnt_model_debug_buffer(m.h, 2, out.ctypes.data_as(C.POINTER(C.c_float)))
    assert n == m.hp.dim
    return out.astype(np.float64)


@pytest.mark.parametrize("name,n,pt", [("tiny_q8", 5, 16), ("tiny_q8", 130, 64), ("tiny_q4sl", 77, 32), ("tiny_q8", 450, 128),
                                       ("tiny_long", 1100, 64)])
def test_paged_residual_follows_the_f16_caches(qb, models, name, n, pt):
    ctx = 2048 if name == "tiny_long" else 512
    m = qb.Model(models(name), ctx_len=ctx)
    try:
        rng = np.random.default_rng(n)
        prompt = rng.integers(0, m.hp.n_tokens, n)
        other = np.concatenate([rng.integers(0, m.hp.n_tokens, n - 1), prompt[-1:]])
        nxt = int(rng.integers(0, m.hp.n_tokens))
        got = {}
        for kind in (F16, PAGED):
            if kind == F16:
                m.batch_init(3, ctx)
            else:
                m.batch_init_paged(3, ctx, 3 * (ctx // pt) + 2, pt)
            m.prefill_batch(1, prompt)
            a = residual(qb, m)
            m.decode_batch([1], [nxt])
            b = residual(qb, m)
            m.prefill_batch(2, other)
            got[kind] = (a, b, residual(qb, m))
        apart = np.linalg.norm(got[F16][0] - got[F16][2])
        assert apart > 0
        for i in range(3):
            assert np.linalg.norm(got[PAGED][i] - got[F16][i]) <= 0.1 * apart, i
    finally:
        m.close()


def test_fork_reset_and_resize(qb, models):
    """Forked sequences answer as their source does, freed pages serve again, and a pool of another size holds the same."""
    m = qb.Model(models("tiny_q8"), ctx_len=512)
    try:
        rng = np.random.default_rng(3)
        prompt = rng.integers(0, m.hp.n_tokens, 75)
        m.batch_init_paged(4, 256, 20, 16)  # 75 positions: 5 pages, the last one part-filled
        first = m.prefill_batch(0, prompt)
        for s in (1, 2, 3):
            m.batch_fork(0, s)  # 4 shared pages, 1 of its own each
        steps, ids = 12, [[first] for _ in range(4)]
        for k in range(steps):
            out = m.decode_batch([0, 1, 2, 3], [i[-1] for i in ids])
            for i, t in zip(ids, out):
                i.append(int(t))
        assert ids[1] == ids[0] and ids[2] == ids[0] and ids[3] == ids[0]
        # 87 positions: 4 shared pages + 4 x 2 = 12 of 20
        m.batch_reset(2)
        with pytest.raises(qb.QntError, match="in use"):
            m.batch_resize(9)
        m.batch_resize(10)
        assert list(m.decode_batch([0, 3], [ids[0][-1]] * 2)) == [int(m.decode_batch([1], [ids[0][-1]])[0])] * 2
        with pytest.raises(qb.QntError, match="no free pages"):
            m.prefill_batch(2, prompt[:17])
        m.batch_resize(14)
        want = m.prefill_batch(2, prompt[:17])  # the refused call left nothing behind
        m.batch_reset(2)
        assert m.prefill_batch(2, prompt[:17]) == want
    finally:
        m.close()


def test_a_decode_step_without_room_changes_nothing(qb, models):
    m = qb.Model(models("tiny_q8"), ctx_len=512)
    try:
        rng = np.random.default_rng(4)
        m.batch_init_paged(2, 128, 3, 16)
        a = m.prefill_batch(0, rng.integers(0, m.hp.n_tokens, 16))
        b = m.prefill_batch(1, rng.integers(0, m.hp.n_tokens, 16))
        with pytest.raises(qb.QntError, match="no free pages"):
            m.decode_batch([0, 1], [a, b])  # needs two pages, one is free
        one = m.decode_batch([0], [a])
        m.batch_resize(6)
        m.decode_batch([1], [b])
        m.batch_reset(1)
        m.batch_fork(0, 1)
        two = m.decode_batch([0, 1], [int(one[0])] * 2)
        assert two[0] == two[1]
    finally:
        m.close()


def test_paged_refusals(qb, models):
    m = qb.Model(models("tiny_q8"), ctx_len=512)
    try:
        for args in ((0, 128, 8, 16), (2, 1, 8, 16), (2, 513, 8, 16), (2, 128, 0, 16), (2, 128, 8, 48), (8193, 128, 8, 16),
                     (2, 128, (1 << 20) + 1, 16)):
            with pytest.raises(qb.QntError):
                m.batch_init_paged(*args)
        m.batch_init(2, 128)
        with pytest.raises(qb.QntError):
            m.batch_fork(0, 1)  # the f16 caches are not paged
        with pytest.raises(qb.QntError):
            m.batch_resize(8)
        m.batch_init_paged(2, 128, 8, 16)
        m.prefill_batch(0, [1, 2, 3])
        m.prefill_batch(1, [1, 2, 3])
        for src, dst in ((0, 1), (0, 0), (0, 2), (-1, 1)):
            with pytest.raises(qb.QntError):
                m.batch_fork(src, dst)
        with pytest.raises(qb.QntError):
            m.decode_batch([0, 0], [4, 5])
        with pytest.raises(qb.QntError):
            m.batch_resize(0)
    finally:
        m.close()
