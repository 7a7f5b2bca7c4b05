"""A call that fails leaves batched serving from the paged 8-bit KV cache as it was: host and device agree about every length."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu


def served(qb, m, rng, spoil):
    """Prompts and steps, with calls of a bad token id in between where `spoil`; the ids, and the pages in use at the end."""
    n = m.hp.n_tokens
    m.batch_init_paged(3, 256, 40, 16)

    def bad(call):
        if spoil:
            with pytest.raises(qb.QntError):
                call()

    prompts = [rng.integers(0, n, k) for k in (30, 16, 33)]
    bad(lambda: m.prefill_batch(0, [1, 2, 10 ** 6, 3]))  # an empty sequence stays empty
    bad(lambda: m.prefill_batch(0, [-1]))
    ids = [[m.prefill_batch(s, p)] for s, p in enumerate(prompts)]
    for k in range(20):
        seqs = [0, 1, 2] if k % 3 else [2, 0]
        bad(lambda: m.decode_batch(seqs, [ids[s][-1] for s in seqs[:-1]] + [10 ** 6]))
        bad(lambda: m.decode_batch(seqs, [-1] + [ids[s][-1] for s in seqs[1:]]))
        bad(lambda: m.prefill_batch(1, list(prompts[0]) + [10 ** 6]))
        for s, t in zip(seqs, m.decode_batch(seqs, [ids[s][-1] for s in seqs])):
            ids[s].append(int(t))
    bad(lambda: m.prefill_batch(1, list(prompts[0]) + [10 ** 6]))
    pages = sum(-(-(len(p) + len(i) - 1) // 16) for p, i in zip(prompts, ids))
    with pytest.raises(qb.QntError, match=f"{pages} pages are in use"):
        m.batch_resize(1)
    for s in range(3):
        m.batch_reset(s)
    m.batch_resize(1)  # every page has come back
    return ids


def test_a_bad_token_id_changes_nothing(qb, models):
    m = qb.Model(models("tiny_q8"), ctx_len=512)
    try:
        want = served(qb, m, np.random.default_rng(7), False)
        assert served(qb, m, np.random.default_rng(7), True) == want
    finally:
        m.close()


def test_a_long_prompt_with_a_bad_token_id_late(qb, models):
    """Of a prompt of several chunks none is taken."""
    m = qb.Model(models("tiny_long"), ctx_len=2048)
    try:
        rng = np.random.default_rng(8)
        prompt = rng.integers(0, m.hp.n_tokens, 1100)
        m.batch_init_paged(2, 2048, 80, 64)
        with pytest.raises(qb.QntError):
            m.prefill_batch(0, list(prompt[:1050]) + [10 ** 6])
        a = m.prefill_batch(0, prompt)
        assert m.prefill_batch(1, prompt) == a
    finally:
        m.close()
